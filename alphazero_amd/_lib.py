"""ctypes binding of libazamd.so (the C ABI declared in include/azamd.h).

The library is the product: there is no Python or CPU fallback for anything it
computes.  Loading fails loudly when the shared object is missing.
"""
import ctypes as C
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("AZAMD_LIB") or os.path.join(_HERE, "libazamd.so")   # AZAMD_LIB: a diagnostic build of the same library


class AzError(RuntimeError):
    pass


class EngineConfig(C.Structure):
    _fields_ = [
        ("n_games", C.c_int32),
        ("c_puct", C.c_double),
        ("dirichlet_alpha", C.c_double),
        ("dirichlet_epsilon", C.c_double),
        ("temperature_threshold", C.c_int32),
        ("pool_nodes_per_game", C.c_int64),
        ("seed", C.c_uint64),
        ("device", C.c_int32),
    ]


class NetConfig(C.Structure):
    _fields_ = [
        ("num_blocks", C.c_int32),
        ("num_filters", C.c_int32),
        ("se_ratio", C.c_int32),
        ("max_batch", C.c_int32),
        ("device", C.c_int32),
    ]


class SelfplayStats(C.Structure):
    _fields_ = [
        ("simulations", C.c_uint64),
        ("nn_evals", C.c_uint64),
        ("moves", C.c_uint64),
        ("games_finished", C.c_uint64),
        ("samples_pending", C.c_uint64),
        ("network_rows", C.c_uint64),
    ]


class NormArgs(C.Structure):
    _fields_ = ([("n", C.c_int64)] + [(k, C.c_int32) for k in ("c", "hw", "hidden", "dtype", "channels_last", "training")]
                + [("eps", C.c_double), ("momentum", C.c_double)]
                + [(k, C.c_void_p) for k in (
                    "x", "residual", "weight", "bias", "running_mean", "running_var", "num_batches", "fc1_weight", "fc1_bias",
                    "fc2_weight", "fc2_bias", "saved", "workspace", "out", "grad", "dx", "dresidual", "dweight", "dbias",
                    "dfc1_weight", "dfc1_bias", "dfc2_weight", "dfc2_bias")])


class LossArgs(C.Structure):
    _fields_ = ([("n", C.c_int64)] + [(k, C.c_int32) for k in ("actions", "outcomes", "dtype")]
                + [(k, C.c_void_p) for k in ("policy", "wl", "target_pi", "target_wl", "mask", "losses", "stats", "up_loss",
                                             "up_pi", "up_wl", "dpolicy", "dwl")]
                + [("grads_ready", C.c_int32)])


class AdamGroup(C.Structure):
    _fields_ = ([(k, C.c_double) for k in ("lr", "beta1", "beta2", "eps", "weight_decay")]
                + [("decoupled", C.c_int32), ("end", C.c_int32)])


class AdamConfig(C.Structure):
    _fields_ = ([("max_norm", C.c_double), ("seed", C.c_uint64), ("state_bits", C.c_int32)]
                + [(k, C.c_void_p) for k in ("pieces", "m", "v", "m_scale", "v_scale", "steps", "norm", "scratch")])


# name -> (argtypes); every entry point returns int (az_adam_plan and az_adam_scratch: int64)
_VP = C.c_void_p
_SIGNATURES = {
    "az_version": [],
    "az_movegen_encode": [C.c_int64, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP],
    "az_engine_create": [C.POINTER(_VP), C.POINTER(EngineConfig)],
    "az_engine_destroy": [_VP],
    "az_engine_set_positions": [_VP, C.c_int32, _VP, _VP, _VP, _VP, _VP, _VP],
    "az_engine_update_positions": [_VP, C.c_int32, _VP, _VP, _VP, _VP, _VP, _VP],
    "az_engine_root_counts": [_VP, _VP, _VP],
    "az_engine_get_positions": [_VP, _VP, _VP, _VP, _VP, _VP],
    "az_engine_set_active": [_VP, _VP, _VP],
    "az_engine_roots_prepare": [_VP, _VP, _VP, _VP],
    "az_engine_roots_expand": [_VP, _VP, _VP],
    "az_engine_add_noise": [_VP, _VP, _VP],
    "az_engine_select": [_VP, _VP, _VP, _VP],
    "az_engine_expand_backup": [_VP, _VP, _VP, _VP],
    "az_engine_node_children": [_VP, C.c_int32, C.c_int64] + [_VP] * 11,
    "az_engine_action_probs": [_VP, _VP, _VP, _VP],
    "az_engine_roots_children": [_VP, C.c_int32] + [_VP] * 12,
    "az_engine_advance": [_VP, _VP, _VP],
    "az_engine_set_root": [_VP, C.c_int32, C.c_int64, _VP],
    "az_engine_set_roots": [_VP, C.c_int32, _VP, _VP, _VP],
    "az_engine_search_leaf_parallel": [_VP, C.c_int32, _VP, C.c_int32, C.c_int32, _VP],
    "az_engine_import_tree": [_VP, C.c_int32, C.c_int32, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP],
    "az_engine_pool_usage": [_VP, _VP, _VP],
    "az_engine_stats": [_VP, _VP, _VP, _VP],
    "az_net_create": [C.POINTER(_VP), C.POINTER(NetConfig)],
    "az_net_destroy": [_VP],
    "az_net_max_batch": [_VP],
    "az_net_load_state": [_VP, _VP, C.c_int64],
    "az_net_forward": [_VP, C.c_int32, _VP, _VP, _VP, _VP, _VP, _VP, _VP],
    "az_net_forward_noalloc": [_VP, C.c_int32, _VP, _VP, _VP, _VP, _VP, _VP, _VP],
    "az_net_forward_planes": [_VP, C.c_int32, _VP, _VP, _VP, _VP, _VP, _VP],
    "az_net_set_timing": [_VP, C.c_int32],
    "az_net_set_tower_form": [_VP, C.c_int32],
    "az_net_debug_stamps": [_VP, _VP, C.c_int32],
    "az_net_tower_time": [_VP, C.POINTER(C.c_double), C.POINTER(C.c_int64)],
    "az_engine_attach_net": [_VP, _VP],
    "az_engine_search": [_VP, C.c_int32, C.c_int32, _VP],
    "az_engine_play_move": [_VP, C.c_int32, C.c_int32, _VP, C.c_int32, _VP],
    "az_engine_chosen_actions": [_VP, _VP, _VP],
    "az_engine_drain_samples": [_VP, C.c_int64, _VP, _VP, _VP, C.POINTER(C.c_int64), _VP],
    "az_engine_drain_packed": [_VP, C.c_int64, _VP, C.POINTER(C.c_int64), _VP],
    "az_unpack_samples": [C.c_int64, _VP, _VP, _VP, _VP, _VP],
    "az_engine_selfplay_stats": [_VP, C.POINTER(SelfplayStats), _VP],
    "az_norm_sizes": [C.POINTER(NormArgs), C.POINTER(C.c_int64)],
    "az_norm_forward": [C.POINTER(NormArgs), _VP],
    "az_norm_backward": [C.POINTER(NormArgs), _VP],
    "az_policy_value_loss_ready": [C.POINTER(LossArgs)],
    "az_policy_value_loss_forward": [C.POINTER(LossArgs), _VP],
    "az_policy_value_loss_backward": [C.POINTER(LossArgs), _VP],
    "az_adam_plan": [C.c_int32, _VP, _VP, _VP],
    "az_adam_scratch": [C.c_int32],
    "az_graph_fill_by_kernels": [_VP, C.POINTER(C.c_int32)],
    "az_adam_step": [C.POINTER(AdamConfig), C.c_int32, C.POINTER(AdamGroup), C.c_int32, _VP, _VP, _VP, _VP],
}
_OPTIONAL = {}

OPTIM_CHUNK, OPTIM_PAD, OPTIM_GROUPS = 4096, 256, 48      # AZ_OPTIM_CHUNK, AZ_OPTIM_PAD, AZ_OPTIM_GROUPS
PACKED_SAMPLE_BYTES = 792     # AZ_PACKED_SAMPLE_BYTES

_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise AzError(
                f"{LIB_PATH} is missing: build it with alphazero_amd/csrc/build.sh "
                "(__graft_entry__.build()).  There is no fallback path.")
        L = C.CDLL(LIB_PATH)
        L.az_last_error.restype = C.c_char_p
        for name, args in _SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = C.c_int64 if name in ("az_adam_plan", "az_adam_scratch") else C.c_int
        for name, args in _OPTIONAL.items():
            if hasattr(L, name):
                fn = getattr(L, name)
                fn.argtypes = args
                fn.restype = C.c_int
        _lib = L
    return _lib


def check(rc):
    if rc != 0:
        raise AzError(f"libazamd error {rc}: {lib().az_last_error().decode()}")


_torch_ops = None


def torch_ops():
    """The native torch side of the training operators (csrc/torch_ops.cpp), calling the library that lib() loaded."""
    global _torch_ops
    if _torch_ops is None:
        L = lib()
        try:
            import torch  # noqa: F401  (the module resolves against torch's libraries)
            from . import _azops
        except ImportError as e:
            raise AzError(f"alphazero_amd/_azops.so does not load ({e}): build it with alphazero_amd/csrc/build.sh "
                          "(__graft_entry__.build()).  There is no fallback path.") from e
        names = ("az_last_error", "az_norm_sizes", "az_norm_forward", "az_norm_backward", "az_policy_value_loss_ready", "az_policy_value_loss_forward",
                 "az_policy_value_loss_backward", "az_adam_plan", "az_adam_scratch", "az_adam_step")
        _azops.bind({n: C.cast(getattr(L, n), C.c_void_p).value for n in names}, AzError)
        _torch_ops = _azops
    return _torch_ops


def exported_symbols():
    """Every symbol include/azamd.h declares (parsed from the header)."""
    import re
    hdr = os.path.join(os.path.dirname(_HERE), "include", "azamd.h")
    text = open(hdr).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(az_[a-z0-9_]+)\s*\(", text)))
