"""distspmm_b200 — B200-native distributed CSR x dense SpMM (the hot path of DistSpMM).

Layers
  include/distspmm.h        C ABI (the drop-in boundary)
  libdistspmm_b200.so       native library: loader, planner, sm_100a kernels, rank runtime
  bin/dist_spmm_node        reference-compatible CLI
  pattern / act / attention sparse layers on one GPU: the product with bias, activation and
                            residual, attention masked by a matrix's entries (with gradients),
                            and attention of single tokens over a cache
  matrix / planner / spmm / dist   Python face of the C ABI (ctypes; torch only supplies
                            device memory, streams and torch.distributed)
  comm_test / fit_comm_model       the bulk-vs-sparse fetch microbenchmark and the
                            selector-model fit (command lines of the reference's tools)
"""
from ._lib import DspError, lib
from .matrix import Csr, dense_b, dense_b_rows, gen_rmat, gen_stencil27, gen_uniform, load_from_csr, load_rows, make_matrix, save_csr
from . import planner
from .planner import hierarchical_iterative_refinement_allocation

__all__ = [
    "DspError", "lib", "Csr", "dense_b", "dense_b_rows", "gen_rmat", "gen_stencil27", "gen_uniform", "load_from_csr", "load_rows",
    "make_matrix", "save_csr", "planner", "hierarchical_iterative_refinement_allocation",
]


_LAZY = {
    "SpmmPlan": "spmm", "SparsePattern": "pattern",
    **dict.fromkeys(("spmm_act", "spmm_act_forward", "spmm_act_backward"), "act"),
    **dict.fromkeys(("sparse_attention", "sparse_attention_forward", "sparse_attention_backward",
                     "sparse_attention_decode"), "attention"),
    **dict.fromkeys(("Rank", "build_local_group", "TorchComm", "distributed_plan", "connect_peers", "make_rank",
                     "global_plan", "fetch_view"), "dist"),
}


def __getattr__(name):
    # torch-dependent modules load on first use
    if name not in _LAZY:
        raise AttributeError(name)
    import importlib
    value = getattr(importlib.import_module("." + _LAZY[name], __name__), name)
    globals()[name] = value
    return value
