"""ctypes binding of libp2n_hip.so (include/p2n.h).

The library is built in-tree by pointcloudsegmentation_amd/csrc/Makefile
(`__graft_entry__.build()`); there is no fallback: a missing or unloadable
library raises, so a GPU path can never silently run on something else.
"""
import ctypes
import os
import subprocess

# One HIP runtime per process: PyTorch ships its own libamdhip64.so.7 and libp2n_hip.so
# NEEDs the same soname, so torch has to be loaded first for the dynamic loader to hand
# our library torch's runtime (a second runtime from /opt/rocm sees no device and does
# not share streams or allocations with torch).
import torch  # noqa: F401  (must precede ctypes.CDLL below)

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libp2n_hip.so")
CSRC = os.path.join(_HERE, "csrc")

_lib = None

c_f = ctypes.c_void_p      # device float*
c_i = ctypes.c_void_p      # device int32*
c_vp = ctypes.c_void_p
c_int = ctypes.c_int
c_sz = ctypes.c_size_t
c_long = ctypes.c_long
c_float = ctypes.c_float

# name -> (restype, argtypes); mirrors include/p2n.h one to one
SIGNATURES = {
    "p2n_version": (c_int, []),
    "p2n_last_error": (ctypes.c_char_p, []),
    "p2n_param_count": (ctypes.c_long, [c_int, c_int]),
    "p2n_packed_param_count": (ctypes.c_long, [c_int, c_int]),
    "p2n_pack_eval_params": (c_int, [c_f, c_int, c_int, c_f, c_vp]),
    "p2n_forward_eval_workspace_bytes": (c_sz, [c_int, c_int, c_int, c_int]),
    "p2n_forward_eval": (c_int, [c_f, c_int, c_int, c_int, c_int, c_f, c_f, c_f, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_forward_eval_noalloc": (c_int, [c_f, c_int, c_int, c_int, c_int, c_f, c_f, c_f, c_f, c_f, c_f, c_vp]),
    "p2n_packed_param_count_bf16": (ctypes.c_long, [c_int, c_int]),
    "p2n_pack_eval_params_bf16": (c_int, [c_f, c_int, c_int, c_f, c_vp]),
    "p2n_forward_eval_bf16": (c_int, [c_f, c_int, c_int, c_int, c_int, c_f, c_f, c_f, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_packed_param_count_x3": (ctypes.c_long, [c_int, c_int]),
    "p2n_pack_eval_params_x3": (c_int, [c_f, c_int, c_int, c_f, c_vp]),
    "p2n_forward_eval_x3_workspace_bytes": (c_sz, [c_int, c_int, c_int, c_int]),
    "p2n_forward_eval_x3": (c_int, [c_f, c_int, c_int, c_int, c_int, c_f, c_f, c_f, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_fps_workspace_bytes": (c_sz, [c_int, c_int, c_int]),
    "p2n_fps_workgroups_per_cloud": (c_int, [c_int, c_int]),
    "p2n_fps_cluster_kind": (c_int, [c_int, c_int]),
    "p2n_fps": (c_int, [c_f, c_int, c_int, c_int, c_int, c_i, c_i, c_vp, c_sz, c_vp]),
    "p2n_ball_query": (c_int, [c_f, c_f, c_int, c_int, c_int, c_float, c_int, c_i, c_vp]),
    "p2n_knn": (c_int, [c_f, c_f, c_int, c_int, c_int, c_int, c_i, c_f, c_vp]),
    "p2n_knn_self_workspace_bytes": (c_sz, [c_int, c_int]),
    "p2n_knn_self": (c_int, [c_f, c_int, c_int, c_int, c_i, c_f, c_vp, c_sz, c_vp]),
    "p2n_group_gather": (c_int, [c_f, c_i, c_int, c_int, c_int, c_int, c_int, c_f, c_vp]),
    "p2n_group_gather_bwd": (c_int, [c_f, c_i, c_int, c_int, c_int, c_int, c_int, c_f, c_vp]),
    "p2n_three_nn": (c_int, [c_f, c_f, c_int, c_int, c_int, c_f, c_i, c_f, c_vp]),
    "p2n_three_interpolate": (c_int, [c_f, c_i, c_f, c_int, c_int, c_int, c_int, c_f, c_vp]),
    "p2n_three_interpolate_bwd": (c_int, [c_f, c_i, c_f, c_int, c_int, c_int, c_int, c_f, c_vp]),
    "p2n_train_workspace_bytes": (c_sz, [c_int, c_int, c_int, c_int]),
    "p2n_train_forward": (c_int, [c_f, c_int, c_int, c_int, c_int, c_vp, c_float, c_f, c_f, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_train_backward": (c_int, [c_f, c_f, c_int, c_int, c_int, c_int, c_vp, c_vp, c_vp, c_sz, c_vp]),
    "p2n_train_forward_bf16": (c_int, [c_f, c_int, c_int, c_int, c_int, c_vp, c_float, c_f, c_f, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_train_backward_bf16": (c_int, [c_f, c_f, c_int, c_int, c_int, c_int, c_vp, c_vp, c_vp, c_sz, c_vp]),
    "p2n_train_forward_x3": (c_int, [c_f, c_int, c_int, c_int, c_int, c_vp, c_float, c_f, c_f, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_train_backward_x3": (c_int, [c_f, c_f, c_int, c_int, c_int, c_int, c_vp, c_vp, c_vp, c_sz, c_vp]),
    "p2n_mlp_train_workspace_bytes": (c_sz, [ctypes.c_long, c_int, c_vp, c_int]),
    "p2n_mlp_train_forward": (c_int, [c_f, ctypes.c_long, c_int, c_vp, c_int, c_vp, c_float, c_f, c_vp, c_sz, c_vp]),
    "p2n_mlp_train_backward": (c_int, [c_f, c_f, ctypes.c_long, c_int, c_vp, c_int, c_vp, c_vp, c_f, c_vp, c_sz, c_vp]),
    "p2n_dense_instances_workspace_bytes": (c_sz, [c_int, c_int]),
    "p2n_dense_instances": (c_int, [c_vp, c_int, c_int, c_int, c_i, c_i, c_i, c_i, c_i, c_vp, c_sz, c_vp]),
    "p2n_combine3": (c_int, [c_f, c_f, c_f, c_f, ctypes.c_long, c_f, c_vp]),
    "p2n_instance_seg_loss_workspace_bytes": (c_sz, [c_int, c_int, c_int, c_int, c_int]),
    "p2n_instance_seg_loss": (c_int, [c_f, c_f, c_i, c_i, c_i, c_i, c_int, c_int, c_int, c_int, c_float, c_float,
                                      c_int, c_f, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_instance_seg_loss_knn": (c_int, [c_f, c_f, c_i, c_i, c_i, c_i, c_i, c_int, c_int, c_int, c_int, c_float, c_float,
                                          c_int, c_f, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_sa_group": (c_int, [c_f, c_f, c_f, c_i, c_int, c_int, c_int, c_int, c_int, c_f, c_vp]),
    "p2n_pointwise_layer_workspace_bytes": (c_sz, [c_int, c_int]),
    "p2n_pointwise_layer": (c_int, [c_f, c_int, c_int, ctypes.c_long, c_f, c_f, c_f, c_int, c_int, c_f, c_vp, c_sz, c_vp]),
    "p2n_group_max": (c_int, [c_f, c_int, c_int, c_int, c_int, c_f, c_vp]),
    "p2n_group_max_cm": (c_int, [c_f, c_int, c_long, c_long, c_int, c_f, c_vp, c_vp]),
    "p2n_group_max_cm_bwd": (c_int, [c_f, c_vp, c_int, c_long, c_int, c_long, c_f, c_vp]),
    "p2n_level_packed_floats": (ctypes.c_long, [c_int, c_int, c_vp, c_int]),
    "p2n_level_pack": (c_int, [c_int, c_int, c_vp, c_vp, c_int, ctypes.c_double, c_f, c_vp]),
    "p2n_sa_level": (c_int, [c_f, c_int, c_f, c_f, c_int, c_i, c_int, c_int, c_int, c_int, c_int, c_vp, c_f, c_f, c_vp]),
    "p2n_fp_level_workspace_bytes": (c_sz, [c_int, c_int, c_int, c_int, c_int, c_vp]),
    "p2n_fp_level": (c_int, [c_i, c_f, c_f, c_f, c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_vp, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_gather_xyz": (c_int, [c_f, c_int, c_i, c_int, c_int, c_int, c_f, c_vp]),
    "p2n_normalize_rows": (c_int, [c_f, ctypes.c_long, c_int, c_f, c_vp]),
    "p2n_cluster_workspace_bytes": (c_sz, [ctypes.c_long, c_int, c_int]),
    "p2n_cluster_embeddings": (c_int, [c_f, ctypes.c_long, c_int, ctypes.c_double, c_int, c_i, c_i, c_vp, c_sz, c_vp]),
    "p2n_cluster_counts": (c_int, [c_vp, ctypes.c_long, c_int, c_int, c_i, c_vp]),
    "p2n_cluster_stats": (c_int, [c_vp, ctypes.c_long, c_int, c_int, c_vp, c_vp]),
    "p2n_preprocess_workspace_bytes": (c_sz, []),
    "p2n_preprocess_points": (c_int, [c_vp, c_vp, ctypes.c_long, c_f, c_vp, c_vp, c_sz, c_vp]),
    "p2n_forward_eval_raw": (c_int, [c_vp, c_vp, c_int, c_int, c_f, c_vp, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_int8_weight_bytes": (c_long, [c_int, c_int]),
    "p2n_int8_pack_weight": (c_int, [c_f, c_f, c_int, c_int, c_f, c_f, c_f, c_f, ctypes.c_double, c_vp, c_vp]),
    "p2n_quantize_tokens": (c_int, [c_vp, c_int, c_long, c_int, c_long, c_vp, c_f, c_vp]),
    "p2n_int8_linear_workspace_bytes": (c_sz, [c_long, c_int, c_int]),
    "p2n_int8_linear": (c_int, [c_vp, c_int, c_long, c_int, c_long, c_vp, c_int, c_int, c_vp, c_vp, c_sz, c_vp]),
    "p2n_int8_mlp": (c_int, [c_f, c_int, c_long, c_int, c_vp, c_vp, c_int, c_int, c_f, c_vp]),
    "p2n_max_of_columns": (c_int, [c_f, c_long, c_int, c_f, c_vp]),
    "p2n_act8_kept_bytes": (c_sz, [c_int, c_int, c_long, c_int]),
    "p2n_act8_workspace_bytes": (c_sz, [c_int, c_int, c_long, c_int]),
    "p2n_act8_forward": (c_int, [c_f, c_int, c_int, c_long, c_f, c_f, c_int, c_f, c_f, c_f, c_f, c_vp, c_float, c_float, c_f,
                                 c_vp, c_sz, c_vp, c_sz, c_vp]),
    "p2n_act8_backward": (c_int, [c_f, c_int, c_int, c_long, c_f, c_int, c_f, c_f, c_int, c_vp, c_sz, c_f, c_f, c_f, c_f, c_f,
                                  c_vp, c_sz, c_vp]),
    "p2n_act8_norm_relu_forward": (c_int, [c_f, c_int, c_int, c_long, c_f, c_f, c_f, c_f, c_vp, c_float, c_float, c_f, c_vp, c_sz,
                                           c_vp, c_sz, c_vp]),
    "p2n_act8_norm_relu_backward": (c_int, [c_f, c_int, c_int, c_long, c_f, c_int, c_vp, c_sz, c_f, c_f, c_f, c_vp, c_sz, c_vp]),
    "p2n_profile_enable": (c_int, [c_int]),
    "p2n_profile_select": (c_int, [c_int]),
    "p2n_profile_collect": (c_int, [c_int, ctypes.POINTER(ctypes.c_float), ctypes.POINTER(ctypes.c_int)]),
}


class P2nError(RuntimeError):
    pass


def build(force: bool = False) -> str:
    """Compile libp2n_hip.so for gfx950 (hipcc cross-compiles without a GPU)."""
    cmd = ["make", "-C", CSRC, "-j8"] + (["-B"] if force else [])
    subprocess.check_call(cmd, stdout=subprocess.DEVNULL)
    return LIB_PATH


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise P2nError(
                f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                "(there is no fallback path for GPU tensors)")
        _lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(_lib, name)   # AttributeError = header/library mismatch: let it propagate
            fn.restype = res
            fn.argtypes = args
    return _lib


def check(rc: int, what: str):
    if rc != 0:
        msg = lib().p2n_last_error().decode(errors="replace")
        if rc == 1:
            raise ValueError(f"{what}: {msg}")
        raise P2nError(f"{what}: rc={rc}: {msg}")
