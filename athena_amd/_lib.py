"""ctypes binding of ``libathena_hip.so`` (declared in ``include/athena_hip.h``).

The library is the product's only compute path: there is no CPU or eager fallback.  A missing
or unloadable library raises at first use with the command that builds it.
"""
import ctypes
import os
import struct
from ctypes import (POINTER, Structure, c_char_p, c_double, c_float, c_int, c_int32, c_int64, c_long,
                    c_size_t, c_uint32, c_uint64, c_void_p)

_HERE = os.path.dirname(os.path.abspath(__file__))
# (ATHENA_HIP_LIB names another build of the library, e.g. to compare two kernels on one machine)
LIB_PATH = os.environ.get("ATHENA_HIP_LIB") or os.path.join(_HERE, "lib", "libathena_hip.so")

F32, BF16 = 0, 1
ACT_NONE, ACT_RELU6, ACT_GELU, ACT_MUL_DGELU, ACT_MUL_DRELU6 = 0, 1, 2, 3, 4
ACT_UNARY, ACT_MUL_DUNARY = 16, 32          # + k: relu elu selu leaky_relu sigmoid softplus softsign tanh relu6


class GemmDesc(Structure):
    """Mirror of ``athena_gemm_desc``."""
    _fields_ = [
        ("A", c_void_p), ("B", c_void_p), ("C", c_void_p), ("C_pre", c_void_p), ("bias", c_void_p),
        ("aux", c_void_p), ("rng_state", c_void_p),
        ("M", c_int32), ("N", c_int32), ("K", c_int32),
        ("trans_a", c_int32), ("trans_b", c_int32),
        ("lda", c_int32), ("ldb", c_int32), ("ldc", c_int32), ("ldaux", c_int32),
        ("in_dtype", c_int32), ("out_dtype", c_int32), ("aux_dtype", c_int32),
        ("act", c_int32), ("accumulate", c_int32), ("split_k", c_int32),
        ("alpha", c_float), ("drop_p", c_float), ("rng_site", c_uint32),
        ("b_colsum", c_void_p), ("workspace", c_void_p), ("workspace_bytes", c_int64),
    ]


class WgradItem(Structure):
    """Mirror of ``athena_wgrad_item``."""
    _fields_ = [
        ("A", c_void_p), ("B", c_void_p), ("C", c_void_p), ("bsum", c_void_p),
        ("M", c_int32), ("N", c_int32), ("K", c_int32),
        ("lda", c_int32), ("ldb", c_int32), ("ldc", c_int32),
        ("first_tile", c_int32), ("tiles_m", c_int32),
    ]


class WgradFold(Structure):
    """Mirror of ``athena_wgrad_fold``."""
    _fields_ = [
        ("dst", c_void_p), ("src", c_void_p), ("n", c_int64), ("part_stride", c_int64),
        ("parts", c_int32), ("first_block", c_int32),
    ]


class LayerTailFwd(Structure):
    """Mirror of ``athena_layer_tail_fwd_desc``."""
    _fields_ = [
        ("rows", c_int32), ("d_model", c_int32), ("dff", c_int32), ("reserved", c_int32),
        ("ctx", c_void_p), ("x", c_void_p), ("wo_t", c_void_p), ("bo", c_void_p), ("gamma1", c_void_p),
        ("beta1", c_void_p), ("w1_t", c_void_p), ("b1", c_void_p), ("w2_t", c_void_p), ("b2", c_void_p),
        ("gamma2", c_void_p), ("beta2", c_void_p),
        ("eps", c_float), ("drop_p", c_float), ("rng_state", c_void_p),
        ("site_res1", c_uint32), ("site_ffn", c_uint32), ("site_res2", c_uint32), ("reserved2", c_uint32),
        ("z1", c_void_p), ("y1", c_void_p), ("mean1", c_void_p), ("rstd1", c_void_p), ("hpre", c_void_p),
        ("h", c_void_p), ("z2", c_void_p), ("y2", c_void_p), ("mean2", c_void_p), ("rstd2", c_void_p),
        ("next_w_t", c_void_p * 3), ("next_b", c_void_p * 3), ("next_out", c_void_p * 3),
        ("x_f32", c_void_p), ("y_out_f32", c_void_p),
    ]


class LayerTailBwd(Structure):
    """Mirror of ``athena_layer_tail_bwd_desc``."""
    _fields_ = [
        ("rows", c_int32), ("d_model", c_int32), ("dff", c_int32), ("reserved", c_int32),
        ("dy", c_void_p), ("z2", c_void_p), ("mean2", c_void_p), ("rstd2", c_void_p), ("gamma2", c_void_p),
        ("hpre", c_void_p), ("w2", c_void_p), ("w1", c_void_p), ("z1", c_void_p), ("mean1", c_void_p),
        ("rstd1", c_void_p), ("gamma1", c_void_p), ("wo", c_void_p),
        ("drop_p", c_float), ("reserved2", c_float), ("rng_state", c_void_p),
        ("site_res1", c_uint32), ("site_ffn", c_uint32), ("site_res2", c_uint32), ("reserved3", c_uint32),
        ("df", c_void_p), ("dh", c_void_p), ("da", c_void_p), ("dx", c_void_p), ("dctx", c_void_p),
        ("slab2", c_void_p), ("slab1", c_void_p),
        ("add_dqkv", c_void_p), ("add_w", c_void_p * 3),
    ]


class AdamCfg(Structure):
    """Mirror of ``athena_adam_cfg``."""
    _fields_ = [
        ("beta1", c_float), ("beta2", c_float), ("eps", c_float), ("clip_norm", c_float),
        ("d_model", c_float), ("warmup_steps", c_float), ("k", c_float), ("decay_steps", c_float),
        ("decay_rate", c_float), ("grad_scale", c_float),
        ("schedule", c_float), ("initial_lr", c_float), ("start_decay_steps", c_float), ("final_lr", c_float),
    ]


# The descriptors of the decoding entry points, packed in one go: a decoding step issues many small calls, and setting
# some thirty Structure fields one by one takes longer than such a kernel runs.  Pointers (0 = null), then
# 64-bit, then 32-bit members, as include/athena_hip.h declares them.
KvPlanDesc = struct.Struct("@12Qq6i")              # athena_kv_plan_desc
Kv8AppendDesc = struct.Struct("@7Q4q8i")           # athena_kv8_append_desc
Kv8AttentionDesc = struct.Struct("@11Q6q12i2f")    # athena_kv8_attention_desc
LogitsDesc = struct.Struct("@11Q7q6i")             # athena_logits_desc

_P = c_void_p
_S = c_void_p   # stream
_SIGNATURES = {
    "athena_last_error": (c_char_p, []),
    "athena_abi_version": (c_int, []),
    "athena_timing_begin": (c_int, []),
    "athena_timing_count": (c_int, []),
    "athena_timing_end": (c_int, []),
    "athena_timing_read": (c_int, [c_int, c_int, POINTER(c_float)]),
    "athena_gemm": (c_int, [POINTER(GemmDesc), _S]),
    "athena_gemm_grouped": (c_int, [POINTER(GemmDesc), c_int, _S]),
    "athena_gemm_wgrad_plan": (c_int, [POINTER(WgradItem), c_int, POINTER(c_int)]),
    "athena_gemm_wgrad_table": (c_int, [_P, c_int, c_int, _S]),
    "athena_gemm_wgrad_split": (c_int, [POINTER(WgradItem), c_int, c_int, _P, c_int64, POINTER(c_int64),
                                        POINTER(WgradItem), c_int, POINTER(c_int), POINTER(WgradFold), c_int,
                                        POINTER(c_int), POINTER(c_int)]),
    "athena_gemm_wgrad_fold": (c_int, [_P, c_int, c_int, _S]),
    "athena_gemm_workspace_bytes": (c_int64, [c_int, c_int, c_int, c_int]),
    "athena_colsum": (c_int, [_P, c_int, c_int, c_int, c_int, _P, _S]),
    "athena_add_layernorm_fwd": (c_int, [_P, _P, _P, _P, c_float, c_int, c_int, c_int, c_float, _P, c_uint32,
                                         _P, _P, _P, _P, _S]),
    "athena_add_layernorm_fwd_wide": (c_int, [_P, _P, _P, _P, _P, c_float, c_int, c_int, c_int, c_float, _P, c_uint32,
                                              _P, _P, _P, _P, _P, _S]),
    "athena_add_layernorm_bwd": (c_int, [_P, _P, _P, _P, _P, c_int, c_int, c_int, c_float, _P, c_uint32, c_int,
                                         _P, _P, _P, _P, _P, c_int64, _S]),
    "athena_add_layernorm_bwd_workspace_bytes": (c_int64, [c_int, c_int]),
    "athena_add_layernorm_bwd_slabs": (c_int, [c_int, c_int]),
    "athena_prepare_labels": (c_int, [_P, _P, _P, c_int, c_int, c_int, c_int, c_int, _P, _P, _P, _P, _P, _S]),
    "athena_ln_fold_batched": (c_int, [_P, c_int, c_int, _S]),
    "athena_mpc_loss_fwd": (c_int, [_P, c_int, _P, _P, _P, c_int, c_int, c_int, _P, _S]),
    "athena_mpc_loss_bwd": (c_int, [_P, c_int, _P, _P, _P, c_int, c_int, c_int, _P, c_float, _P, c_int, _S]),
    "athena_layer_tail_workgroups": (c_int, [c_int]),
    "athena_layer_tail_fwd": (c_int, [POINTER(LayerTailFwd), _S]),
    "athena_layer_tail_bwd": (c_int, [POINTER(LayerTailBwd), _S]),
    "athena_mha_fwd": (c_int, [_P, _P, _P, c_int, c_int, c_int, _P, c_int, c_int, c_int, c_int, c_int, c_int,
                               c_int, c_float, _P, c_int, _P, _S]),
    "athena_mha_bwd": (c_int, [_P, _P, _P, c_int, c_int, c_int, _P, c_int, c_int, c_int, c_int, c_int, c_int,
                               c_int, c_float, _P, _P, c_int, _P, _P, _P, _P, _P, c_int, c_int, c_int, _S]),
    "athena_mha_weights": (c_int, [_P, _P, c_int, c_int, _P, c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_float, _P, _S]),
    "athena_conv3x3s2_fwd": (c_int, [_P, _P, c_int, _P, c_int, c_int, c_int, c_int, c_int, c_int, _P, _S]),
    "athena_conv3x3s2_dgrad": (c_int, [_P, _P, _P, c_int, c_int, c_int, c_int, c_int, c_int, _P, _S]),
    "athena_conv1_moments_len": (c_int64, []),
    "athena_conv1_bn_stats": (c_int, [_P, _P, c_int, c_int, c_int, c_int, _P, _P, _S]),
    "athena_conv1_bn_relu6_fwd": (c_int, [_P, _P, _P, _P, _P, _P, c_float, c_int, c_int, c_int, c_int, c_int, c_int,
                                          _P, _S]),
    "athena_conv1_bn_bwd_workspace_bytes": (c_int64, [c_int]),
    "athena_conv1_bn_bwd": (c_int, [_P, _P, _P, _P, _P, _P, _P, _P, c_int, c_int, c_int, c_int, c_int, _P, c_int64, _P, _P,
                                    _P, _S]),
    "athena_conv3x3s2_wgrad": (c_int, [_P, _P, _P, c_int, c_int, c_int, c_int, c_int, c_int, _P, c_int64, _S]),
    "athena_conv3x3s2_wgrad_workspace_bytes": (c_int64, [c_int, c_int, c_int, c_int, c_int, c_int]),
    "athena_conv3x3s2_small_cin_fwd": (c_int, [_P, _P, _P, c_int, c_int, c_int, c_int, c_int, c_int, _P, _S]),
    "athena_conv3x3s2_small_cin_wgrad": (c_int, [_P, _P, _P, c_int, c_int, c_int, c_int, c_int, c_int, _S]),
    "athena_bn_finalize": (c_int, [_P, c_long, c_int, c_float, c_float, _P, _P, _P, _S]),
    "athena_bn_relu6_apply": (c_int, [_P, _P, _P, _P, c_long, c_int, c_int, _P, _S]),
    "athena_bn_relu6_infer": (c_int, [_P, _P, _P, _P, _P, c_float, c_long, c_int, c_int, _P, _S]),
    "athena_bn_relu6_bwd_scratch_bytes": (c_int64, [c_long, c_int]),
    "athena_bn_relu6_bwd": (c_int, [_P, _P, _P, _P, _P, c_long, c_int, c_int, _P, c_int64, _P, _P, _P, _S]),
    "athena_bn_colstats": (c_int, [_P, c_long, c_int, c_int, _P, _S]),
    "athena_bn_apply": (c_int, [_P, _P, _P, _P, c_long, c_int, c_int, _P, _S]),
    "athena_bn_infer": (c_int, [_P, _P, _P, _P, _P, c_float, c_long, c_int, c_int, _P, _S]),
    "athena_bn_bwd": (c_int, [_P, _P, _P, _P, _P, c_long, c_int, c_int, _P, c_int64, _P, _P, _P, _S]),
    "athena_conv2d_out_shape": (c_int, [c_int, c_int, c_int, c_int, c_int, c_int, POINTER(c_int), POINTER(c_int)]),
    "athena_conv2d_fwd": (c_int, [_P, _P, _P] + [c_int] * 10 + [_P, _S]),
    "athena_conv2d_dgrad": (c_int, [_P, _P, _P] + [c_int] * 10 + [_P, _S]),
    "athena_conv2d_wgrad_workspace_bytes": (c_int64, [c_int] * 10),
    "athena_conv2d_wgrad": (c_int, [_P, _P, _P] + [c_int] * 10 + [_P, c_int64, _S]),
    "athena_im2col": (c_int, [_P, c_int, _P, c_int, c_int] + [c_int] * 8 + [_S]),
    "athena_rnn_workspace_bytes": (c_int64, [c_int, c_int, c_int]),
    "athena_rnn_fwd": (c_int, [c_int, _P, _P, _P, _P, _P, _P, _P, _P, _P, c_int, c_int, c_int, c_int, _P, c_int64, _S]),
    "athena_rnn_bwd": (c_int, [c_int, _P, _P, _P, _P, _P, _P, _P, _P, c_int, c_int, c_int, c_int, _P, c_int64, _S]),
    "athena_add_pe_dropout": (c_int, [_P, _P, c_int, c_int, c_int, c_int, c_float, c_float, _P, c_uint32, _P, _S]),
    "athena_dropout_bwd": (c_int, [_P, c_long, c_int, c_float, c_float, _P, c_uint32, _P, _P, _S]),
    "athena_embed_fwd": (c_int, [_P, _P, _P, c_int, c_int, c_int, c_int, c_int, c_float, c_float, _P, c_uint32,
                                 _P, _S]),
    "athena_embed_bwd": (c_int, [_P, _P, c_int, c_int, c_int, c_int, c_int, c_float, c_float, _P, c_uint32, _P, _S]),
    "athena_ctc_workspace_bytes": (c_size_t, [c_int, c_int, c_int]),
    "athena_ctc_loss_fwd": (c_int, [_P, c_int, c_int, _P, _P, _P, c_int, c_int, c_int, c_int, c_int, _P, _P, _P,
                                    c_size_t, _S]),
    "athena_ctc_loss_fwd_static": (c_int, [_P, c_int, c_int, _P, _P, _P, c_int, c_int, c_int, c_int, c_int, _P, _P, _S]),
    "athena_ctc_loss_bwd": (c_int, [_P, c_int, c_int, _P, _P, _P, c_int, c_int, c_int, c_int, c_int, _P, c_float,
                                    _P, c_int, _P, c_size_t, _S]),
    "athena_ctc_loss_fwd_bwd": (c_int, [_P, c_int, c_int, _P, _P, _P, c_int, c_int, c_int, c_int, c_int, _P, _P, c_float,
                                        _P, c_int, _P, c_size_t, _S]),
    "athena_rescale_unless": (c_int, [_P, c_long, c_int, _P, c_float, _S]),
    "athena_ce_loss_fwd": (c_int, [_P, c_int, c_int, _P, c_int, c_int, c_float, _P, _P, _S]),
    "athena_ce_loss_bwd": (c_int, [_P, c_int, c_int, _P, c_int, c_int, c_float, _P, _P, c_float, _P, c_int, _S]),
    "athena_group_sum": (c_int, [_P, c_int, c_int, c_float, _P, _S]),
    "athena_weighted_sum": (c_int, [_P, _P, c_int, _P, _S]),
    "athena_panel_gemm": (c_int, [_P, c_long, c_int, c_int, _P, _P, _P, _P, _S]),
    "athena_panel_gemm_k": (c_int, [_P, c_long, c_int, c_int, c_int, _P, _P, _P, c_int, c_int, _P, c_long, _S]),
    "athena_argmax_rows": (c_int, [_P, c_int, c_int, c_int, c_int, _P, _S]),
    "athena_seq_errors": (c_int, [_P, c_int, _P, _P, c_int, c_int, c_int, c_int, c_int, _P, _P, _S]),
    "athena_clip_adam_step": (c_int, [_P, _P, _P, _P, c_long, _P, c_int, _P, _P, POINTER(AdamCfg), _P, _S]),
    "athena_refresh_shadows": (c_int, [_P, _P, _P, c_int, _P, c_long, _S]),
    "athena_advance_rng": (c_int, [_P, _S]),
    "athena_cast": (c_int, [_P, c_int, _P, c_int, c_long, _S]),
    "athena_copy_many": (c_int, [_P, _P, _P, c_int, _S]),
    "athena_axpby": (c_int, [c_float, _P, c_float, _P, c_long, c_int, _S]),
    "athena_kv_plan": (c_int, [c_char_p, _S]),
    "athena_kv8_append": (c_int, [c_char_p, _S]),
    "athena_kv8_attention_workspace_bytes": (c_int64, [c_char_p]),
    "athena_kv8_attention": (c_int, [c_char_p, _S]),
    "athena_logits_process": (c_int, [c_char_p, _S]),
}

EXPORTED_SYMBOLS = tuple(_SIGNATURES)

_lib = None


def load():
    """Load the shared library once; raise with build instructions if it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            "athena_amd: %s is missing. Build it with `python -c 'import __graft_entry__ as g; g.build()'` "
            "or athena_amd/csrc/build.sh; there is no fallback path." % LIB_PATH)
    lib = ctypes.CDLL(LIB_PATH)
    for name, (res, args) in _SIGNATURES.items():
        fn = getattr(lib, name)     # AttributeError names the missing symbol
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def check(rc, what):
    if rc != 0:
        msg = load().athena_last_error()
        raise RuntimeError("%s failed (%d): %s" % (what, rc, msg.decode() if msg else ""))
