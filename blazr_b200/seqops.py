"""Python harness over the C ABI of libb200seq.so (include/b200seq.h): dense bfloat16-weight linear layers and the sequence
operators of layer-list models (stream mixing + grouped RMS norm, carried-state causal convolutions, chunk / window attention
over a paged KV pool, the state-space recurrence, gated activations, the depth-averaged residual, mixtures of experts, retention,
latent attention, per-head projections, token shift + gated post-norm, the branch sum + output norm of two-branch mixers, the bigram
embedding, PolyNorm, soft caps, differential attention, minGRU and real-gated linear recurrences, soft-max routing with identity experts,
the delta rule with per-channel decays, layers normed on both sides with sinusoidal positions and a token-dependent addition, the selective scan
with a decay per channel and state, the residual of parallel layers, a KV cache held in 4 bits and its attention, page copies, sampling rules, drafts
verified, the weight of cached keys and their eviction, arg-max).

Like blazr_b200/ops.py, PyTorch is plumbing only (device memory, streams); every compute call goes through ctypes.  The library
is compiled on first use when it is missing (`ensure_built`): a fresh checkout needs nothing but nvcc.  There is no CPU
fallback: without the library or without an sm_100 GPU the calls raise.
"""
from __future__ import annotations

import ctypes as C
import fcntl
import os
import shutil
import subprocess
from itertools import chain
from struct import error as StructError, pack
from typing import Optional, Sequence, Tuple

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
SRC_DIR = os.path.join(_HERE, "csrc", "seq")
LIB_PATH = os.environ.get("B200SEQ_LIB") or os.path.join(_HERE, "lib", "libb200seq.so")

F32, BF16 = 0, 2
CONV_RESIDUAL, CONV_SILU = 1, 2
ACT_SWISH_CLAMP, ACT_GELU_TANH, ACT_RELU2, ACT_IDENT = 0, 1, 2, 3   # gated: clamped swish, tanh-gelu gate; plain: squared relu, the product itself
ACT_GELU_ERF, ACT_TANH = 4, 5                                       # plain: exact gelu, tanh
ACT_NONE = -1
ACT_KINDS = {"swish_clamp": ACT_SWISH_CLAMP, "gelu_tanh": ACT_GELU_TANH, "relu2": ACT_RELU2, "gelu_erf": ACT_GELU_ERF, "tanh": ACT_TANH}
ACT_GATED = (ACT_SWISH_CLAMP, ACT_GELU_TANH)
PATH_AUTO, PATH_ROWS, PATH_TILED, PATH_TC = 0, 1, 2, 3
TC_MIN_ROWS = 32   # b200seq_linear's automatic choice takes the tensor-core path from this many rows
_DT = {torch.float32: F32, torch.bfloat16: BF16}

EXPORTS = ["b200seq_last_error", "b200seq_version", "b200seq_launch_count", "b200seq_error_flags", "b200seq_embed_streams", "b200seq_hc_norm", "b200seq_hc_norm_conv",
           "b200seq_causal_conv", "b200seq_group_rmsnorm", "b200seq_gated_act", "b200seq_linear", "b200seq_linear_gated", "b200seq_attn_prep", "b200seq_attn", "b200seq_attn_scratch_floats",
           "b200seq_ssm_scan", "b200seq_ssm_scratch_floats", "b200seq_argmax", "b200seq_linear_act", "b200seq_act", "b200seq_depth_norm", "b200seq_attn_prep_ex",
           "b200seq_attn_ex", "b200seq_moe_route", "b200seq_moe_sort", "b200seq_moe_linear", "b200seq_moe_gather", "b200seq_moe_combine", "b200seq_moe_router", "b200seq_moe_table_route", "b200seq_moe_linear_act", "b200seq_head_linear", "b200seq_latent_gather",
           "b200seq_latent_prep", "b200seq_rotary", "b200seq_retention", "b200seq_retention_scratch_floats", "b200seq_token_shift", "b200seq_post_norm",
           "b200seq_moe_route_ex", "b200seq_moe_router_ex", "b200seq_moe_combine_ex", "b200seq_causal_conv_ex", "b200seq_embed_bigram", "b200seq_branch_norm", "b200seq_polynorm", "b200seq_softcap",
           "b200seq_diff_combine", "b200seq_min_gru", "b200seq_rg_lru", "b200seq_delta", "b200seq_delta_scratch_floats", "b200seq_embed_pos", "b200seq_sandwich_norm",
           "b200seq_token_gate", "b200seq_side_close", "b200seq_linear_silu", "b200seq_moe_route_rule", "b200seq_moe_router_rule", "b200seq_retention_partials",
           "b200seq_selective_scan", "b200seq_scan_scratch_floats", "b200seq_parallel_close", "b200seq_kv4_page_bytes", "b200seq_kv4_store", "b200seq_kv4_load",
           "b200seq_attn_prep_kv4", "b200seq_attn_kv4", "b200seq_attn_kv4_scratch_floats", "b200seq_copy_pages", "b200seq_process_logits",
           "b200seq_verify_drafts", "b200seq_verify_scratch_bytes", "b200seq_key_weights", "b200seq_key_weights_scratch_floats", "b200seq_evict_keys"]

# argument types of the operators' C entries (include/b200seq.h): p pointer, i int, l int64, z size_t, f float.  Declared, plain numbers are converted by ctypes
# as they are passed; an object made for each of them and a stream object looked up for each call took half of a call's 4 - 8 us.
_ARG = dict(p=C.c_void_p, i=C.c_int, l=C.c_int64, z=C.c_size_t, f=C.c_float)
SIGNATURES = {
    "error_flags": "p", "embed_streams": "ppfiiipp", "hc_norm": "pppppiiifpipip", "hc_norm_conv": "pppppiiifpppipip", "causal_conv": "plppppiiipilp",
    "group_rmsnorm": "plpiiifpip", "gated_act": "pliifffipip", "linear": "pilpiiiplip", "linear_silu": "pilpiiipliiip", "linear_gated": "pilpiiifffpilp",
    "attn_prep": "plpppiiiifp", "attn": "plpppiiiifiiipipzp", "ssm_scan": "pliiplpppppiiiippzp", "linear_act": "pilpiiiifffpilp", "act": "pliiifffpilp",
    "depth_norm": "plippppppifpppippip", "attn_prep_ex": "plppppppp", "attn_ex": "plpppppppipzp", "latent_prep": "pliiplpiiiipfpfpplpip",
    "latent_gather": "plpiipip", "head_linear": "pilpiiiiipillp", "rotary": "pliiipiipffp", "retention_partials": "iiii", "retention": "plppppipzp",
    "token_shift": "pipppppip", "post_norm": "ppplpfppfipippipppppp", "moe_route": "pliiiiipppp", "moe_router": "pilpiiiiiiiplppp", "moe_table_route": "ppiiipppp",
    "moe_sort": "piippppp", "moe_linear": "pilippppiiiiipilp", "moe_linear_act": "pilippppiiiiifffpilp", "moe_gather": "plpiiiplp", "moe_combine": "pppiiipplpp",
    "moe_route_ex": "pliiiiiippppp", "moe_router_ex": "pilpiiiiiiiipplppp", "moe_route_rule": "plippppp", "moe_router_rule": "pilpiiipplppp",
    "moe_combine_ex": "ppppipiiipplpp", "causal_conv_ex": "plpppppiiipilpilp", "embed_bigram": "pppppfiiiippip", "branch_norm": "ppppfppfpfipippipp",
    "polynorm": "pliipfpilp", "softcap": "plfp", "diff_combine": "piiiifffpip", "min_gru": "pliiipppipip", "rg_lru": "plplppfplipppiipip", "delta": "plppplppipzp",
    "embed_pos": "pppfpippppfpip", "sandwich_norm": "pppfppipippipp", "token_gate": "pliiplippip", "side_close": "pppfpppliippppipippipp",
    "selective_scan": "piplpplppppipzp", "parallel_close": "pp", "argmax": "piipp", "kv4_page_bytes": "iii", "kv4_store": "plplipiiiippp", "kv4_load": "pppiiiiplplp",
    "attn_prep_kv4": "plppppp", "attn_kv4": "plpppppipzip", "attn_kv4_scratch_floats": "ppi", "copy_pages": "ppiipip", "process_logits": "pliippipppppiplplp",
    "verify_scratch_bytes": "iii", "verify_drafts": "pliipippppppplpppzp", "key_weights_scratch_floats": "ppii", "key_weights": "plpppipiliipzp",
    "evict_keys": "pppiiiiiiiilpppippiiiiipp"
}


class SeqError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"b200seq error {code}: {msg}")
        self.code = code


class StepDesc(C.Structure):
    """b200seq_step: device pointers of one step's int32 arrays (see include/b200seq.h)"""
    _fields_ = [("tok_ent", C.c_void_p), ("tok_pos", C.c_void_p), ("ent_start", C.c_void_p), ("ent_slot", C.c_void_p), ("ent_pos0", C.c_void_p),
                ("block_table", C.c_void_p), ("T", C.c_int32), ("B", C.c_int32), ("max_blocks", C.c_int32), ("block_size", C.c_int32)]


class AttnDesc(C.Structure):
    """b200seq_attn_desc: sizes, columns of the projection row and mask / rotation constants of one attention layer"""
    _fields_ = [("H", C.c_int32), ("G", C.c_int32), ("D", C.c_int32), ("V", C.c_int32), ("q_col", C.c_int32), ("k_col", C.c_int32), ("v_col", C.c_int32),
                ("gate_col", C.c_int32), ("scale", C.c_float), ("chunk", C.c_int32), ("window", C.c_int32), ("pool", C.c_int32), ("qk_eps", C.c_float),
                ("rot_dims", C.c_int32), ("rot_freq", C.c_void_p), ("rot_scale", C.c_float), ("sink", C.c_void_p), ("latent_v", C.c_int32), ("gate", C.c_void_p), ("gate_ld", C.c_int64), ("ctx_rows", C.c_int32), ("kd", C.c_int32), ("kv_ld", C.c_int64), ("krot", C.c_void_p), ("krot_ld", C.c_int64),
                ("q_norm_w", C.c_void_p), ("k_norm_w", C.c_void_p), ("norm_full", C.c_int32), ("rot_half", C.c_int32), ("in_bias", C.c_void_p), ("kv_shared", C.c_int32),
                ("vg", C.c_int32), ("softcap", C.c_float), ("head_scale", C.c_void_p), ("keep_first", C.c_int32), ("gate_elem", C.c_int32), ("rot_pos", C.c_void_p)]


class RetentionDesc(C.Structure):
    """b200seq_retention_desc: sizes, columns of the projection row, decays and rotation constants of one retention layer"""
    _fields_ = [("H", C.c_int32), ("D", C.c_int32), ("V", C.c_int32), ("q_col", C.c_int32), ("k_col", C.c_int32), ("v_col", C.c_int32), ("g_col", C.c_int32),
                ("decay", C.c_void_p), ("eps", C.c_float), ("rot_dims", C.c_int32), ("rot_half", C.c_int32), ("rot_freq", C.c_void_p), ("rot_scale", C.c_float),
                ("k_scale", C.c_float), ("norm_w", C.c_void_p), ("gate_sigmoid", C.c_int32), ("sumsq", C.c_void_p)]


def retention_desc(H: int, D: int, V: int, decay: torch.Tensor, eps: float, k_scale: float, *, rot_freq: Optional[torch.Tensor] = None, rot_half: bool = True,
                   rot_scale: float = 1.0, norm_w: Optional[torch.Tensor] = None, gate_sigmoid: bool = False) -> "RetentionDesc":
    """descriptor for a projection row laid out q | k | v | gate; decay: device f32 [2, H] (decays, their base-2 logarithms); norm_w: f32 [H * V], one
    norm over all heads, deferred (see include/b200seq.h); the caller keeps the tensors alive"""
    assert decay.dtype == torch.float32 and tuple(decay.shape) == (2, H) and decay.is_contiguous()
    d = RetentionDesc(H, D, V, 0, H * D, 2 * H * D, 2 * H * D + H * V, decay.data_ptr(), eps, 2 * rot_freq.numel() if rot_freq is not None else 0, int(rot_half),
                      rot_freq.data_ptr() if rot_freq is not None else None, rot_scale, k_scale, norm_w.data_ptr() if norm_w is not None else None, int(gate_sigmoid))
    assert norm_w is None or (norm_w.dtype == torch.float32 and norm_w.numel() == H * V and norm_w.is_contiguous())
    d.width = 2 * H * D + 2 * H * V
    return d


class DeltaDesc(C.Structure):
    """b200seq_delta_desc: sizes, columns of the projection row, weights and constants of one delta-rule layer"""
    _fields_ = [("H", C.c_int32), ("D", C.c_int32), ("V", C.c_int32), ("r_col", C.c_int32), ("k_col", C.c_int32), ("v_col", C.c_int32), ("g_col", C.c_int32),
                ("a_col", C.c_int32), ("w_col", C.c_int32), ("rank", C.c_int32), ("w2", C.c_void_p), ("w0", C.c_void_p), ("a_b", C.c_void_p), ("norm_w", C.c_void_p),
                ("decay_scale", C.c_float), ("unit_eps", C.c_float), ("eps", C.c_float)]


def delta_desc(H: int, D: int, V: int, rank: int, w2: torch.Tensor, w0: torch.Tensor, a_b: torch.Tensor, norm_w: torch.Tensor, decay_scale: float, unit_eps: float,
               eps: float) -> "DeltaDesc":
    """descriptor for a projection row laid out r | k | v | gate | removal logits | low rank; w2 bf16 [H * D, rank], the vectors f32; the caller keeps the tensors alive"""
    assert w2.dtype == torch.bfloat16 and w2.is_contiguous() and tuple(w2.shape) == (H * D, rank)
    assert all(t.dtype == torch.float32 and t.numel() == n for t, n in ((w0, H * D), (a_b, H * D), (norm_w, H * V)))
    cols = [0, H * D, 2 * H * D, 2 * H * D + H * V, 2 * H * (D + V), 3 * H * D + 2 * H * V]
    d = DeltaDesc(H, D, V, *cols, rank, w2.data_ptr(), w0.data_ptr(), a_b.data_ptr(), norm_w.data_ptr(), decay_scale, unit_eps, eps)
    d.width = cols[-1] + rank
    return d


def attn_desc(H: int, G: int, D: int, V: int, scale: float, *, values_from_keys: bool = False, gated: bool = True, chunk: int = 0, window: int = 0, pool: int = 0,
              qk_eps: float = -1.0, rot_freq: Optional[torch.Tensor] = None, rot_scale: float = 1.0, sink: Optional[torch.Tensor] = None,
              q_norm_w: Optional[torch.Tensor] = None, k_norm_w: Optional[torch.Tensor] = None, norm_full: bool = False, rot_half: bool = False,
              in_bias: Optional[torch.Tensor] = None, kv_shared: bool = False, value_heads: int = 0, softcap: float = 0.0, head_scale: Optional[torch.Tensor] = None,
              keep_first: int = 0, gate_elem: bool = False) -> "AttnDesc":
    """descriptor for a projection row laid out q | k | v | gate (v absent when the values are the keys, k and v absent when they are another
    layer's (kv_shared), gate absent when not gated); value_heads: number of value heads when it is not G.
    Device tensors (rot_freq f32 [rot_dims / 2], sink / head_scale f32 [H], norm weights, in_bias f32 [row width]) are kept alive by the caller."""
    Gv = value_heads if value_heads > 0 else G
    k_col = H * D
    v_col = k_col if values_from_keys else k_col + G * D
    end = k_col if kv_shared else v_col + (G * D if values_from_keys else Gv * V)
    ptr = lambda t: t.data_ptr() if t is not None else None
    d = AttnDesc(H, G, D, V, 0, k_col, v_col, end if gated else -1, scale, chunk, window, pool, qk_eps, 2 * rot_freq.numel() if rot_freq is not None else 0,
                 ptr(rot_freq), rot_scale, ptr(sink), 0)
    d.q_norm_w, d.k_norm_w, d.norm_full, d.rot_half, d.in_bias = ptr(q_norm_w), ptr(k_norm_w), int(norm_full), int(rot_half), ptr(in_bias)
    d.kv_shared, d.vg, d.softcap, d.head_scale, d.keep_first = int(kv_shared), (Gv if Gv != G else 0), softcap, ptr(head_scale), keep_first
    d.gate_elem = int(gate_elem and gated)
    d.width = end + ((H * V if gate_elem else H) if gated else 0)
    return d


def expanded_attn_desc(H: int, Dn: int, Rd: int, V: int, scale: float, krot: torch.Tensor, *, gated: bool = True, sink: Optional[torch.Tensor] = None) -> "AttnDesc":
    """descriptor of the attend step of a latent-attention layer over per-head keys and values that were projected out of the step's gathered
    context: rows [H * Dn keys | H * V values]; the Rd rotated key dimensions of every head come from krot, a view [rows, Rd] of the paged pool"""
    D = Dn + Rd
    d = AttnDesc(H, H, D, V, 0, 0, H * Dn, 0 if gated else -1, scale, 0, 0, 0, -1.0, 0, None, 1.0, sink.data_ptr() if sink is not None else None, 0, None, 0,
                 1, Dn if Rd > 0 else 0, H * (Dn + V), krot.data_ptr() if Rd > 0 else None, krot.stride(-2) if Rd > 0 else 0)
    d.width = H * D
    return d


def latent_attn_desc(H: int, R: int, Rd: int, scale: float, *, gated: bool = True, sink: Optional[torch.Tensor] = None) -> "AttnDesc":
    """descriptor of the attend step of a latent-attention layer: H query heads of size R + Rd (latent-space query | rotated part) in rows
    [H * (R + Rd)] (gate logits: the `gate` argument of attn_ex) over ONE key head [c | kr] whose values are its first R floats; no rotation here (b200seq_latent_prep did it)"""
    D = R + Rd
    d = AttnDesc(H, 1, D, R, 0, 0, 0, 0 if gated else -1, scale, 0, 0, 0, -1.0, 0, None, 1.0, sink.data_ptr() if sink is not None else None, 1)
    d.width = H * D
    return d


def _stale() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    srcs = [os.path.join(SRC_DIR, f) for f in os.listdir(SRC_DIR) if f.endswith((".cu", ".cuh"))] + [os.path.join(_HERE, "..", "include", "b200seq.h")]
    return any(os.path.getmtime(s) > t for s in srcs if os.path.exists(s))


def ensure_built(force: bool = False) -> str:
    """compile libb200seq.so (nvcc, sm_100a) if it is missing or older than its sources; safe against concurrent callers"""
    if "B200SEQ_LIB" in os.environ or not (force or _stale()):
        return LIB_PATH
    os.makedirs(os.path.dirname(LIB_PATH), exist_ok=True)
    with open(os.path.join(os.path.dirname(LIB_PATH), ".seq_build.lock"), "w") as lk:
        fcntl.flock(lk, fcntl.LOCK_EX)
        if force or _stale():
            env = dict(os.environ)
            if "NVCC" not in env and shutil.which("nvcc") is None:
                for cand in (os.path.join(env.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc"), "/usr/local/cuda/bin/nvcc"):
                    if os.path.exists(cand):
                        env["NVCC"] = cand
                        break
            r = subprocess.run(["make", "-C", SRC_DIR, "-j8"], capture_output=True, text=True, env=env)
            if r.returncode != 0:
                raise SeqError(-3, "libb200seq build failed:\n" + r.stdout[-3000:] + r.stderr[-3000:])
    return LIB_PATH


_lib = None
VERSION = 2      # of the structs above (include/b200seq.h)


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        ensure_built()
        L = C.CDLL(LIB_PATH)
        if L.b200seq_version() != VERSION:
            raise SeqError(-1, f"{LIB_PATH} is of version {L.b200seq_version()}, its structs are not those of version {VERSION}")
        L.b200seq_last_error.restype = C.c_char_p
        L.b200seq_launch_count.restype = C.c_int64
        L.b200seq_kv4_page_bytes.restype = C.c_int64
        L.b200seq_attn_kv4_scratch_floats.restype = C.c_size_t
        L.b200seq_verify_scratch_bytes.restype = L.b200seq_key_weights_scratch_floats.restype = C.c_size_t
        for name, args in SIGNATURES.items():
            getattr(L, "b200seq_" + name).argtypes = [_ARG[a] for a in args]
        _lib = L
    return _lib


def _check(rc: int):
    if rc != 0:
        raise SeqError(rc, lib().b200seq_last_error().decode())


def _st(t: torch.Tensor) -> int:
    dev = t.device
    if dev.type != "cuda":
        raise ValueError(f"Expected a cuda device, but got: {dev}")
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def launch_count() -> int:
    return int(lib().b200seq_launch_count())


def error_flags() -> int:
    f = C.c_int(0)
    _check(lib().b200seq_error_flags(C.byref(f)))
    return f.value


def _rows2d(t: torch.Tensor):
    shape, strides = t.shape, t.stride()
    assert len(shape) == 2 and strides[1] == 1, "row-major 2-D view expected"
    return shape[0], shape[1], strides[0]


# ---- per-operator timeline (bench / profiling aid): set `timeline = []` and every operator call appends
#      (name, shapes of its positional tensor arguments, positional scalars, start event, end event, keyword arguments as shapes /
#      scalars); None (default) costs nothing ------------------------------------------------------------------------------------
timeline = None


def _timed(fn):
    name = fn.__name__

    def wrap(*a, **k):
        tl = timeline
        if tl is None:
            return fn(*a, **k)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        r = fn(*a, **k)
        e1.record()
        shapes = tuple((tuple(t.shape), t.element_size()) if isinstance(t, torch.Tensor) else None for t in a)
        scal = tuple(t for t in a if isinstance(t, (int, float, bool)))
        kw = {n: ((tuple(t.shape), t.element_size()) if isinstance(t, torch.Tensor) else t) for n, t in k.items() if isinstance(t, (torch.Tensor, int, float, bool))}
        tl.append((name, shapes, scal, e0, e1, kw))
        return r

    wrap.__name__, wrap.__doc__ = name, fn.__doc__
    return wrap


# ---- operators (all arguments are device tensors; outputs are written in place) --------------------------------------------
@_timed
def embed_streams(table: torch.Tensor, ids: torch.Tensor, scale: float, X: torch.Tensor):
    T, S, W = X.shape
    _check(lib().b200seq_embed_streams(_p(table), _p(ids), scale, T, S, W, _p(X), _st(X)))


@_timed
def hc_norm(X: torch.Tensor, y: Optional[torch.Tensor], post: Optional[torch.Tensor], in_w: Optional[torch.Tensor], norm_w: Optional[torch.Tensor],
            groups: int, eps: float, out: Optional[torch.Tensor], rows: Optional[torch.Tensor] = None):
    T, S, W = X.shape
    R = T if rows is None else rows.numel()
    _check(lib().b200seq_hc_norm(_p(X), _p(y), _p(post), _p(in_w), _p(norm_w), S, W, groups, eps, _p(rows), R, _p(out), _DT[out.dtype] if out is not None else F32, _st(X)))


@_timed
def hc_norm_conv(X: torch.Tensor, y: Optional[torch.Tensor], post: Optional[torch.Tensor], in_w: torch.Tensor, norm_w: torch.Tensor, groups: int, eps: float,
                 conv_w: torch.Tensor, conv_state: torch.Tensor, step: "StepDesc", out: torch.Tensor):
    """hc_norm followed by the residual carried convolution in one kernel; only for steps in which every entry brings one token"""
    T, S, W = X.shape
    _check(lib().b200seq_hc_norm_conv(_p(X), _p(y), _p(post), _p(in_w), _p(norm_w), S, W, groups, eps, _p(conv_w), _p(conv_state), C.byref(step),
                                      conv_w.shape[1], _p(out), _DT[out.dtype], _st(X)))


@_timed
def causal_conv(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], state: Optional[torch.Tensor], step: "StepDesc", mode: int, out: torch.Tensor):
    T, Cn, ldx = _rows2d(x)
    _, _, ldo = _rows2d(out)
    _check(lib().b200seq_causal_conv(_p(x), ldx, _p(w), _p(bias), _p(state), C.byref(step), Cn, w.shape[1], mode, _p(out), _DT[out.dtype],
                                     ldo, _st(x)))


@_timed
def group_rmsnorm(x: torch.Tensor, w: Optional[torch.Tensor], groups: int, eps: float, out: torch.Tensor):
    T, D, ldx = _rows2d(x)
    assert out.is_contiguous()
    _check(lib().b200seq_group_rmsnorm(_p(x), ldx, _p(w), T, D, groups, eps, _p(out), _DT[out.dtype], _st(x)))


@_timed
def gated_act(gu: torch.Tensor, limit: float, alpha: float, up_shift: float, out: torch.Tensor, interleaved: bool = False):
    T, F2, ldg = _rows2d(gu)
    assert out.is_contiguous() and out.shape[1] * 2 == F2
    _check(lib().b200seq_gated_act(_p(gu), ldg, T, F2 // 2, limit, alpha, up_shift, int(interleaved), _p(out), _DT[out.dtype], _st(gu)))


@_timed
def linear(x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, path: int = PATH_AUTO, silu: tuple = (0, 0)):
    """y[M, N] (f32) = x[M, K] . w[N, K]^T; w bf16 contiguous; the columns silu[0] .. silu[1] - 1 of y pass silu"""
    M, K, ldx = _rows2d(x)
    _, N, ldy = _rows2d(y)
    assert w.dtype == torch.bfloat16 and w.is_contiguous() and tuple(w.shape) == (N, K) and y.dtype == torch.float32 and y.shape[0] == M
    _check(lib().b200seq_linear_silu(_p(x), _DT[x.dtype], ldx, _p(w), M, N, K, _p(y), ldy, silu[0], silu[1], path, _st(x)))


@_timed
def linear_gated(x: torch.Tensor, w_il: torch.Tensor, limit: float, alpha: float, up_shift: float, out: torch.Tensor):
    """out[M, F] = gated_act(x . w_il^T); w_il bf16 [2F, K] with alternating gate / up rows (up to 8 rows: any activation type;
    more: the tensor-core path, bf16 activations only)"""
    M, K, ldx = _rows2d(x)
    _, F, ldo = _rows2d(out)
    assert w_il.dtype == torch.bfloat16 and w_il.is_contiguous() and tuple(w_il.shape) == (2 * F, K) and out.shape[0] == M
    _check(lib().b200seq_linear_gated(_p(x), _DT[x.dtype], ldx, _p(w_il), M, F, K, limit, alpha, up_shift, _p(out),
                                      _DT[out.dtype], ldo, _st(x)))


@_timed
def linear_act(x: torch.Tensor, w: torch.Tensor, act: int, out: torch.Tensor, limit: float = 0.0, alpha: float = 0.0, shift: float = 0.0):
    """out = act(x . w^T) in one kernel; w bf16 [N, K]; gated kinds (rows of w alternate gate / up) give out [M, N / 2], plain kinds [M, N]
    (up to 8 rows: any activation type; more: the tensor-core path, bf16 activations only)"""
    M, K, ldx = _rows2d(x)
    _, F, ldo = _rows2d(out)
    N = w.shape[0]
    assert w.dtype == torch.bfloat16 and w.is_contiguous() and w.shape[1] == K and out.shape[0] == M and F == (N // 2 if act in ACT_GATED else N)
    _check(lib().b200seq_linear_act(_p(x), _DT[x.dtype], ldx, _p(w), M, N, K, act, limit, alpha, shift, _p(out),
                                    _DT[out.dtype], ldo, _st(x)))


@_timed
def act(z: torch.Tensor, kind: int, out: torch.Tensor, limit: float = 0.0, alpha: float = 0.0, shift: float = 0.0):
    """the same activation on a product that is in memory (z f32 [T, N]; gated kinds read interleaved pairs)"""
    T, N, ldz = _rows2d(z)
    _, _, ldo = _rows2d(out)
    _check(lib().b200seq_act(_p(z), ldz, T, N, kind, limit, alpha, shift, _p(out), _DT[out.dtype], ldo, _st(z)))


@_timed
def depth_norm(x_cur: torch.Tensor, out1: Optional[torch.Tensor], w1: Optional[torch.Tensor], eps: float, *, out2: Optional[torch.Tensor] = None,
               w2: Optional[torch.Tensor] = None, y1: Optional[torch.Tensor] = None, y2: Optional[torch.Tensor] = None, hist: Optional[torch.Tensor] = None,
               n_prev: int = 0, dwa: Optional[torch.Tensor] = None, hist_out: Optional[torch.Tensor] = None, x_out: Optional[torch.Tensor] = None,
               rows: Optional[torch.Tensor] = None):
    """residual sum of a parallel layer (x_cur + (y1 + y2)), learned average over the results of all layers so far (hist [>= n_prev, cap, W] holds the
    earlier ones, dwa [n_prev + 1]), and up to two weighted layer norms of the outcome; rows: only these token rows (outputs are row-compact)"""
    W = x_cur.shape[-1]
    R = x_cur.shape[0] if rows is None else rows.numel()
    o = out1 if out1 is not None else out2
    _check(lib().b200seq_depth_norm(_p(hist), hist.stride(0) if hist is not None else 0, n_prev, _p(dwa), _p(x_cur), _p(y1), _p(y2), _p(hist_out), _p(x_out), W,
                                    eps, _p(w1), _p(w2), _p(rows), R, _p(out1), _p(out2), _DT[o.dtype] if o is not None else F32, _st(x_cur)))


@_timed
def attn_prep_ex(proj: torch.Tensor, step: "StepDesc", d: "AttnDesc", kpool: Optional[torch.Tensor], vpool: Optional[torch.Tensor],
                 kpooled: Optional[torch.Tensor] = None, vpooled: Optional[torch.Tensor] = None, rot_pos: Optional[torch.Tensor] = None):
    """rot_pos: int32 [T], the positions by which q and k turn, where the step's count cached rows"""
    _, _, ld = _rows2d(proj)
    if rot_pos is not None:
        d = _turned("attn_prep_ex", step, d, rot_pos)
    _check(lib().b200seq_attn_prep_ex(_p(proj), ld, C.byref(step), C.byref(d), _p(kpool), _p(vpool), _p(kpooled), _p(vpooled), _st(proj)))


def _turned(name: str, step: "StepDesc", d: "AttnDesc", rot_pos: torch.Tensor) -> "AttnDesc":
    if rot_pos.dtype != torch.int32 or rot_pos.numel() < step.T or not rot_pos.is_contiguous():
        raise ValueError(f"{name}: rot_pos is contiguous int32 of {step.T} positions, not {rot_pos.dtype} {tuple(rot_pos.shape)}")
    d2 = AttnDesc.from_buffer_copy(d)
    d2.rot_pos = rot_pos.data_ptr()
    return d2


@_timed
def attn_ex(proj: torch.Tensor, step: "StepDesc", d: "AttnDesc", kpool: torch.Tensor, vpool: Optional[torch.Tensor], out: torch.Tensor,
            scratch: Optional[torch.Tensor] = None, kpooled: Optional[torch.Tensor] = None, vpooled: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None):
    """gate: f32 [T, H] view (row stride free) of the gate logits when they do not lie in the query rows (d.gate_col is then only a flag)"""
    _, _, ld = _rows2d(proj)
    if gate is not None:        # the descriptor of a call is a copy: the layer's own stays as it was
        d2 = AttnDesc.from_buffer_copy(d)
        d2.gate, d2.gate_ld = gate.data_ptr(), gate.stride(0)
        d = d2
    assert out.is_contiguous() and (scratch is None or (scratch.dtype == torch.float32 and scratch.is_contiguous()))
    _check(lib().b200seq_attn_ex(_p(proj), ld, C.byref(step), C.byref(d), _p(kpool), _p(vpool), _p(kpooled), _p(vpooled), _p(out), _DT[out.dtype], _p(scratch),
                                 scratch.numel() if scratch is not None else 0, _st(proj)))


@_timed
def moe_route(z: torch.Tensor, E: int, groups: int, keep: int, top: int, ids: torch.Tensor, wts: torch.Tensor, counts: Optional[torch.Tensor]):
    """z f32 [T, >= E] router logits -> ids int32 [T, top], wts f32 [T, top], counts int32 [E]"""
    T, _, ldz = _rows2d(z)
    assert ids.dtype == torch.int32 and wts.dtype == torch.float32 and ids.is_contiguous() and wts.is_contiguous() and ids.numel() >= T * top
    _check(lib().b200seq_moe_route(_p(z), ldz, T, E, groups, keep, top, _p(ids), _p(wts), _p(counts), _st(z)))


@_timed
def moe_router(x: torch.Tensor, w: torch.Tensor, E: int, groups: int, keep: int, top: int, z: torch.Tensor, ids: torch.Tensor, wts: torch.Tensor):
    """router projection (all rows of the stacked weight, into z) and the choice among the first E, for at most 8 tokens, in one kernel"""
    T, K, ldx = _rows2d(x)
    _, NR, ldz = _rows2d(z)
    assert w.dtype == torch.bfloat16 and w.is_contiguous() and tuple(w.shape) == (NR, K) and z.dtype == torch.float32 and z.shape[0] == T
    _check(lib().b200seq_moe_router(_p(x), _DT[x.dtype], ldx, _p(w), T, NR, K, E, groups, keep, top, _p(z), ldz, _p(ids), _p(wts), _st(x)))


@_timed
def moe_table_route(table: torch.Tensor, tok_ids: torch.Tensor, T: int, E: int, top: int, ids: torch.Tensor, wts: torch.Tensor, counts: Optional[torch.Tensor]):
    """ids[t][j] = table[tok_ids[t]][j], wts = 1 / top: the experts of a token are a row of a table indexed by its token id"""
    assert table.dtype == torch.int32 and table.is_contiguous() and table.shape[1] == top and tok_ids.dtype == torch.int32 and ids.numel() >= T * top
    _check(lib().b200seq_moe_table_route(_p(table), _p(tok_ids), T, E, top, _p(ids), _p(wts), _p(counts), _st(table)))


@_timed
def moe_sort(ids: torch.Tensor, pairs: int, E: int, counts: torch.Tensor, offs: torch.Tensor, order: torch.Tensor, slot_of: torch.Tensor):
    _check(lib().b200seq_moe_sort(_p(ids), pairs, E, _p(counts), _p(offs), _p(order), _p(slot_of), _st(ids)))


@_timed
def moe_linear(x: torch.Tensor, x_div: int, w: torch.Tensor, ids: torch.Tensor, order: Optional[torch.Tensor], offs: Optional[torch.Tensor], pairs: int, act: int,
               out: torch.Tensor, limit: float = 0.0, alpha: float = 0.0, shift: float = 0.0):
    """one projection of every (token, choice) pair through its expert's weight; w bf16 [E, N, K]; out [pairs, N] (f32 when act is ACT_NONE);
    gated kinds: the rows of every expert's weight alternate (gate j, up j) and out is [pairs, N / 2]"""
    _, K, ldx = _rows2d(x)
    _, No, ldo = _rows2d(out)
    E, N = w.shape[0], w.shape[1]
    assert w.dtype == torch.bfloat16 and w.is_contiguous() and w.shape[2] == K and out.shape[0] >= pairs and No == (N // 2 if act in ACT_GATED else N)
    _check(lib().b200seq_moe_linear_act(_p(x), _DT[x.dtype], ldx, x_div, _p(w), _p(ids), _p(order), _p(offs), pairs, E, N, K, act, limit,
                                        alpha, shift, _p(out), _DT[out.dtype], ldo, _st(x)))


@_timed
def head_linear(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor, ocol: int, act: int = ACT_NONE):
    """out[t, h * ocol + n] = w[h, n] . x[t, h * K : (h + 1) * K] for every head: x [T, >= H * K] rows, w bf16 [H, N, K], out [T, >= (H - 1) * ocol + N] rows
    (f32 when act is ACT_NONE, else a plain kind - ACT_IDENT: the product itself - in out's type)"""
    T, _, ldx = _rows2d(x)
    _, _, ldo = _rows2d(out)
    H, N, K = w.shape
    assert w.dtype == torch.bfloat16 and w.is_contiguous() and out.shape[0] == T and (act != ACT_NONE or out.dtype == torch.float32)
    _check(lib().b200seq_head_linear(_p(x), _DT[x.dtype], ldx, _p(w), T, H, N, K, act, _p(out), _DT[out.dtype], ldo, ocol, _st(x)))


@_timed
def moe_gather(x: torch.Tensor, x_div: int, order: torch.Tensor, pairs: int, out: torch.Tensor):
    """out[r] = x[order[r] // x_div]: the tokens' bf16 activations in the sorted order of their pairs"""
    _, K, ldx = _rows2d(x)
    _, _, ldo = _rows2d(out)
    assert x.dtype == torch.bfloat16 and out.dtype == torch.bfloat16 and out.shape[0] >= pairs and out.shape[1] == K
    _check(lib().b200seq_moe_gather(_p(x), ldx, _p(order), x_div, pairs, K, _p(out), ldo, _st(x)))


@_timed
def moe_combine(ys: torch.Tensor, wts: torch.Tensor, slot_of: Optional[torch.Tensor], T: int, top: int, shared: Optional[torch.Tensor], gate_z: Optional[torch.Tensor],
                y: torch.Tensor):
    W = y.shape[1]
    assert ys.is_contiguous() and y.is_contiguous() and (shared is None or shared.is_contiguous())
    _check(lib().b200seq_moe_combine(_p(ys), _p(wts), _p(slot_of), T, top, W, _p(shared), _p(gate_z), gate_z.stride(0) if gate_z is not None else 0, _p(y), _st(y)))


def tc_usable(x: torch.Tensor, K: int) -> bool:
    """whether the tensor-core path takes this activation matrix (bf16, K % 8 == 0, rows 16-byte aligned)"""
    return x.dtype == torch.bfloat16 and K % 8 == 0 and x.stride(0) % 8 == 0 and x.data_ptr() % 16 == 0


@_timed
def attn_prep(qkvg: torch.Tensor, step: "StepDesc", kpool: torch.Tensor, vpool: torch.Tensor, H: int, G: int, D: int, V: int, qk_eps: float):
    _, _, ld = _rows2d(qkvg)
    _check(lib().b200seq_attn_prep(_p(qkvg), ld, C.byref(step), _p(kpool), _p(vpool), H, G, D, V, qk_eps, _st(qkvg)))


def attn_scratch_floats(T: int, B: int, H: int, G: int, V: int, max_keys: int) -> int:
    """floats of work area the key-split path wants for a step of T tokens (0: the step fills the GPU without splitting)"""
    f = lib().b200seq_attn_scratch_floats
    f.restype = C.c_size_t
    return int(f(T, B, H, G, V, max_keys))


@_timed
def attn(qkvg: torch.Tensor, step: "StepDesc", kpool: torch.Tensor, vpool: torch.Tensor, H: int, G: int, D: int, V: int, scale: float, chunk: int,
         window: int, gated: bool, out: torch.Tensor, scratch: Optional[torch.Tensor] = None):
    _, _, ld = _rows2d(qkvg)
    assert out.is_contiguous() and (scratch is None or (scratch.dtype == torch.float32 and scratch.is_contiguous()))
    _check(lib().b200seq_attn(_p(qkvg), ld, C.byref(step), _p(kpool), _p(vpool), H, G, D, V, scale, chunk, window, int(gated),
                              _p(out), _DT[out.dtype], _p(scratch), scratch.numel() if scratch is not None else 0, _st(qkvg)))


@_timed
def latent_prep(proj: torch.Tensor, c_col: int, gate_col: int, q: torch.Tensor, step: "StepDesc", H: int, Dn: int, Rd: int, R: int, norm_w: torch.Tensor, eps: float,
                rot_freq: Optional[torch.Tensor], rot_scale: float, kpool: torch.Tensor, Qp: Optional[torch.Tensor], qn: Optional[torch.Tensor]):
    """Qp and qn None: the rotated part of every query head turns in place in q (the step attends over per-head keys)"""
    _, _, ldp = _rows2d(proj)
    _, _, ldq = _rows2d(q)
    ldQ = _rows2d(Qp)[2] if Qp is not None else 0
    assert (qn is None or qn.is_contiguous()) and kpool.is_contiguous() and kpool.shape[-1] == R + Rd
    _check(lib().b200seq_latent_prep(_p(proj), ldp, c_col, gate_col, _p(q), ldq, C.byref(step), H, Dn, Rd, R, _p(norm_w), eps,
                                     _p(rot_freq), rot_scale, _p(kpool), _p(Qp), ldQ, _p(qn), _DT[qn.dtype] if qn is not None else F32, _st(proj)))


@_timed
def latent_gather(kpool: torch.Tensor, step: "StepDesc", R: int, ctx_rows: int, out: torch.Tensor):
    """out[r] = the latent (first R floats) of the r-th (entry, position) of the step's contexts, from the paged pool, in out's type"""
    assert kpool.is_contiguous() and out.is_contiguous() and out.shape[0] >= ctx_rows and out.shape[1] == R
    _check(lib().b200seq_latent_gather(_p(kpool), kpool.shape[-1], C.byref(step), R, ctx_rows, _p(out), _DT[out.dtype], _st(kpool)))


@_timed
def rotary(x: torch.Tensor, col: int, nheads: int, D: int, step: "StepDesc", rot_freq: Optional[torch.Tensor], half: bool, rot_scale: float = 1.0, mult: float = 1.0):
    _, _, ld = _rows2d(x)
    _check(lib().b200seq_rotary(_p(x), ld, col, nheads, D, C.byref(step), 2 * rot_freq.numel() if rot_freq is not None else 0, int(half), _p(rot_freq),
                                rot_scale, mult, _st(x)))


def retention_scratch_floats(T: int, B: int, H: int, D: int, V: int) -> int:
    """floats of work area a retention step of T tokens in B entries wants (0: every entry brings one token)"""
    f = lib().b200seq_retention_scratch_floats
    f.restype = C.c_size_t
    return int(f(T, B, H, D, V))


def retention_partials(T: int, B: int, H: int, V: int) -> int:
    """sums of squares a retention step with one norm over all heads leaves per token"""
    return int(lib().b200seq_retention_partials(T, B, H, V))


@_timed
def retention(proj: torch.Tensor, step: "StepDesc", d: "RetentionDesc", state: torch.Tensor, out: torch.Tensor, scratch: Optional[torch.Tensor] = None,
              sumsq: Optional[torch.Tensor] = None):
    """sumsq: f32 [T, retention_partials] of a descriptor with one norm over all heads"""
    _, _, ld = _rows2d(proj)
    if sumsq is not None:       # the descriptor of a call is a copy: the layer's own stays as it was
        assert sumsq.dtype == torch.float32 and sumsq.is_contiguous() and sumsq.numel() >= step.T * retention_partials(step.T, step.B, d.H, d.V)
        d2 = RetentionDesc.from_buffer_copy(d)
        d2.sumsq = sumsq.data_ptr()
        d = d2
    assert out.is_contiguous() and state.is_contiguous() and (scratch is None or (scratch.dtype == torch.float32 and scratch.is_contiguous()))
    _check(lib().b200seq_retention(_p(proj), ld, C.byref(step), C.byref(d), _p(state), _p(out), _DT[out.dtype], _p(scratch),
                                   scratch.numel() if scratch is not None else 0, _st(proj)))


@_timed
def token_shift(x: torch.Tensor, mu: torch.Tensor, state: torch.Tensor, step: "StepDesc", out_plain: Optional[torch.Tensor], out_shift: torch.Tensor):
    T, W = x.shape
    assert x.is_contiguous() and out_shift.is_contiguous() and (out_plain is None or (out_plain.is_contiguous() and out_plain.dtype == out_shift.dtype))
    _check(lib().b200seq_token_shift(_p(x), W, _p(mu), _p(state), C.byref(step), _p(out_plain), _p(out_shift), _DT[out_shift.dtype], _st(x)))


@_timed
def post_norm(x: torch.Tensor, w: torch.Tensor, b: Optional[torch.Tensor], eps: float, *, y: Optional[torch.Tensor] = None, zg: Optional[torch.Tensor] = None,
              gate_b: Optional[torch.Tensor] = None, alpha: float = 1.0, rows: Optional[torch.Tensor] = None, x_out: Optional[torch.Tensor] = None,
              a_out: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None, next_mu: Optional[torch.Tensor] = None,
              next_state: Optional[torch.Tensor] = None, a_shift_out: Optional[torch.Tensor] = None, step: Optional["StepDesc"] = None):
    """layer norm (weight, bias) after the gated residual sum: LN(alpha * x + sigmoid(zg + gate_b) * y); see include/b200seq.h"""
    W = x.shape[-1]
    R = x.shape[0] if rows is None else rows.numel()
    o = a_out if a_out is not None else a_shift_out
    assert x.is_contiguous() and (y is None or y.is_contiguous())
    _check(lib().b200seq_post_norm(_p(x), _p(y), _p(zg), zg.stride(0) if zg is not None else 0, _p(gate_b), alpha, _p(w), _p(b), eps, W,
                                   _p(rows), R, _p(x_out), _p(a_out), _DT[o.dtype] if o is not None else F32, _p(state_out), _p(next_mu), _p(next_state), _p(a_shift_out),
                                   C.byref(step) if step is not None else None, _st(x)))


def ssm_scratch_floats(T: int, B: int, H: int, V: int, N: int) -> int:
    """floats of work area the segmented (parallel over time) scan wants for a step of T tokens in B entries; 0: none needed"""
    f = lib().b200seq_ssm_scratch_floats
    f.restype = C.c_size_t
    return int(f(T, B, H, V, N))


@_timed
def ssm_scan(proj: torch.Tensor, z0: int, dt0: int, xbc: torch.Tensor, A_log: torch.Tensor, Dp: torch.Tensor, dt_bias: torch.Tensor, state: torch.Tensor,
             step: "StepDesc", H: int, V: int, N: int, G: int, out: torch.Tensor, scratch: Optional[torch.Tensor] = None):
    _, _, ldp = _rows2d(proj)
    _, _, ldx = _rows2d(xbc)
    assert out.is_contiguous() and (scratch is None or (scratch.dtype == torch.float32 and scratch.is_contiguous()))
    _check(lib().b200seq_ssm_scan(_p(proj), ldp, z0, dt0, _p(xbc), ldx, _p(A_log), _p(Dp), _p(dt_bias), _p(state), C.byref(step),
                                  H, V, N, G, _p(out), _p(scratch), scratch.numel() if scratch is not None else 0, _st(proj)))


@_timed
def argmax(logits: torch.Tensor, ids: torch.Tensor):
    R, V = logits.shape
    assert logits.is_contiguous() and ids.dtype == torch.int32
    _check(lib().b200seq_argmax(_p(logits), R, V, _p(ids), _st(logits)))


# ---- layers with the norm on the sublayer's output, two-branch mixers, gated linear recurrences ----------------------------------------------
ROUTE_SIGMOID, ROUTE_SOFTMAX, ROUTE_TOP_SOFTMAX = 0, 1, 2


@_timed
def moe_route_ex(z: torch.Tensor, E: int, groups: int, keep: int, top: int, kind: int, correction: Optional[torch.Tensor], ids: torch.Tensor, wts: torch.Tensor,
                 counts: Optional[torch.Tensor]):
    """moe_route with the score kind (ROUTE_SIGMOID / ROUTE_SOFTMAX over the E logits / ROUTE_TOP_SOFTMAX over the chosen ones) and a correction f32 [E] that enters the choice only"""
    T, _, ldz = _rows2d(z)
    assert ids.dtype == torch.int32 and wts.dtype == torch.float32 and ids.is_contiguous() and wts.is_contiguous() and ids.numel() >= T * top
    assert correction is None or (correction.dtype == torch.float32 and correction.numel() == E)
    _check(lib().b200seq_moe_route_ex(_p(z), ldz, T, E, groups, keep, top, kind, _p(correction), _p(ids), _p(wts), _p(counts), _st(z)))


@_timed
def moe_router_ex(x: torch.Tensor, w: torch.Tensor, E: int, groups: int, keep: int, top: int, kind: int, correction: Optional[torch.Tensor], z: torch.Tensor,
                  ids: torch.Tensor, wts: torch.Tensor):
    """moe_router (projection and choice of at most 8 tokens in one kernel) with the score kind and correction of moe_route_ex"""
    T, K, ldx = _rows2d(x)
    _, NR, ldz = _rows2d(z)
    assert w.dtype == torch.bfloat16 and w.is_contiguous() and tuple(w.shape) == (NR, K) and z.dtype == torch.float32 and z.shape[0] == T
    _check(lib().b200seq_moe_router_ex(_p(x), _DT[x.dtype], ldx, _p(w), T, NR, K, E, groups, keep, top, kind, _p(correction), _p(z), ldz, _p(ids),
                                       _p(wts), _st(x)))


@_timed
def moe_combine_ex(ys: torch.Tensor, wts: torch.Tensor, slot_of: Optional[torch.Tensor], ids: torch.Tensor, E_real: int, x_id: torch.Tensor, T: int, top: int,
                   shared: Optional[torch.Tensor], gate_z: Optional[torch.Tensor], y: torch.Tensor):
    """moe_combine where a pair whose expert id is >= E_real is an identity expert: its output is the token's row of x_id (f32 [T, W])"""
    W = y.shape[1]
    assert ys.is_contiguous() and y.is_contiguous() and (shared is None or shared.is_contiguous()) and x_id.is_contiguous() and x_id.dtype == torch.float32
    _check(lib().b200seq_moe_combine_ex(_p(ys), _p(wts), _p(slot_of), _p(ids), E_real, _p(x_id), T, top, W, _p(shared), _p(gate_z),
                                        gate_z.stride(0) if gate_z is not None else 0, _p(y), _st(y)))


@_timed
def causal_conv_ex(x: torch.Tensor, in_bias: Optional[torch.Tensor], w: torch.Tensor, bias: Optional[torch.Tensor], state: Optional[torch.Tensor], step: "StepDesc",
                   mode: int, out: torch.Tensor, out2: Optional[torch.Tensor] = None):
    """causal_conv over x + in_bias (mode 0: convolution + bias, nothing else); out2: a second copy of the result in its own type"""
    T, Cn, ldx = _rows2d(x)
    _, _, ldo = _rows2d(out)
    ldo2 = _rows2d(out2)[2] if out2 is not None else 0
    _check(lib().b200seq_causal_conv_ex(_p(x), ldx, _p(in_bias), _p(w), _p(bias), _p(state), C.byref(step), Cn, w.shape[1], mode, _p(out), _DT[out.dtype],
                                        ldo, _p(out2), _DT[out2.dtype] if out2 is not None else F32, ldo2, _st(x)))


@_timed
def embed_bigram(table: torch.Tensor, bigram: Optional[torch.Tensor], ids: torch.Tensor, ent_prev: torch.Tensor, step: "StepDesc", scale: float, buckets: int,
                 mul_prev: int, mul_cur: int, x: torch.Tensor, a: Optional[torch.Tensor]):
    """x[t] = table[ids[t]] * scale + bigram[hash(previous token, token)] (the last row of bigram at position 0); a: the same in its own type"""
    W = x.shape[-1]
    assert table.dtype == torch.bfloat16 and table.is_contiguous() and x.is_contiguous() and x.dtype == torch.float32 and (a is None or a.is_contiguous())
    assert bigram is None or (bigram.dtype == torch.bfloat16 and bigram.is_contiguous() and tuple(bigram.shape) == (buckets + 1, W))
    _check(lib().b200seq_embed_bigram(_p(table), _p(bigram), _p(ids), _p(ent_prev), C.byref(step), scale, buckets, mul_prev, mul_cur, W, _p(x), _p(a),
                                      _DT[a.dtype] if a is not None else F32, _st(x)))


@_timed
def branch_norm(x: torch.Tensor, y1: torch.Tensor, w: torch.Tensor, eps: float, *, bias1: Optional[torch.Tensor] = None, w_b1: Optional[torch.Tensor] = None, s1: float = 1.0,
                y2: Optional[torch.Tensor] = None, w_b2: Optional[torch.Tensor] = None, s2: float = 1.0, rows: Optional[torch.Tensor] = None,
                x_out: Optional[torch.Tensor] = None, a_out: Optional[torch.Tensor] = None, fin_w: Optional[torch.Tensor] = None):
    """x + rms_norm(s1 * b1 + s2 * b2) * w with b1 = y1 + bias1 (rms-normed with w_b1 when given), b2 = y2 (rms-normed with w_b2); see include/b200seq.h"""
    W = x.shape[-1]
    R = x.shape[0] if rows is None else rows.numel()
    assert x.is_contiguous() and y1.is_contiguous() and (y2 is None or y2.is_contiguous()) and (a_out is None or a_out.is_contiguous())
    _check(lib().b200seq_branch_norm(_p(x), _p(y1), _p(bias1), _p(w_b1), s1, _p(y2), _p(w_b2), s2, _p(w), eps, W, _p(rows), R, _p(x_out),
                                     _p(a_out), _DT[a_out.dtype] if a_out is not None else F32, _p(fin_w), _st(x)))


@_timed
def polynorm(z: torch.Tensor, coef: torch.Tensor, eps: float, out: torch.Tensor):
    """out = c0 N(z) + c1 N(z^2) + c2 N(z^3) + c3 per row, N = division by the root mean square; coef device f32 [4]"""
    T, F, ldz = _rows2d(z)
    _, _, ldo = _rows2d(out)
    assert coef.dtype == torch.float32 and coef.numel() == 4 and out.shape[1] == F
    _check(lib().b200seq_polynorm(_p(z), ldz, T, F, _p(coef), eps, _p(out), _DT[out.dtype], ldo, _st(z)))


@_timed
def softcap(x: torch.Tensor, cap: float):
    assert x.is_contiguous() and x.dtype == torch.float32
    _check(lib().b200seq_softcap(_p(x), x.numel(), cap, _st(x)))


@_timed
def diff_combine(a: torch.Tensor, H: int, G: int, V: int, lam: float, out_scale: float, eps: float, out: torch.Tensor):
    """a f32 [T, 2 * H * V], the two maps per head in the order [key group][map][head of the group] -> out [T, H * V] = unit_rms(a1 - lam * a2) * out_scale"""
    T = a.shape[0]
    assert a.is_contiguous() and a.dtype == torch.float32 and a.shape[1] == 2 * H * V and out.is_contiguous() and tuple(out.shape) == (T, H * V)
    _check(lib().b200seq_diff_combine(_p(a), T, H, G, V, lam, out_scale, eps, _p(out), _DT[out.dtype], _st(a)))


@_timed
def min_gru(proj: torch.Tensor, z_col: int, x_col: int, g_col: int, bias: Optional[torch.Tensor], state: torch.Tensor, step: "StepDesc", Cn: int, out: torch.Tensor):
    _, _, ldp = _rows2d(proj)
    assert out.is_contiguous() and out.shape[1] == Cn and state.is_contiguous() and state.shape[1] == Cn
    _check(lib().b200seq_min_gru(_p(proj), ldp, z_col, x_col, g_col, _p(bias), _p(state), C.byref(step), Cn, _p(out), _DT[out.dtype], _st(proj)))


@_timed
def rg_lru(u: torch.Tensor, gates: torch.Tensor, gate_bias: Optional[torch.Tensor], sp_lam: torch.Tensor, decay_c: float, proj: torch.Tensor, y_col: int,
           bias: Optional[torch.Tensor], state: torch.Tensor, step: "StepDesc", blocks: int, out: torch.Tensor):
    _, Cn, ldu = _rows2d(u)
    _, _, ldg = _rows2d(gates)
    _, _, ldp = _rows2d(proj)
    assert out.is_contiguous() and out.shape[1] == Cn and state.is_contiguous() and state.shape[1] == Cn and sp_lam.numel() == Cn
    _check(lib().b200seq_rg_lru(_p(u), ldu, _p(gates), ldg, _p(gate_bias), _p(sp_lam), decay_c, _p(proj), ldp, y_col, _p(bias),
                                _p(state), C.byref(step), Cn, blocks, _p(out), _DT[out.dtype], _st(proj)))


# ---- delta rule; layers normed on both sides of every sublayer ---------------------------------------------------------------------------------
def delta_scratch_floats(T: int, B: int, H: int, D: int, V: int) -> int:
    """floats of work area a delta-rule step of T tokens in B entries wants (0: every entry brings one token)"""
    f = lib().b200seq_delta_scratch_floats
    f.restype = C.c_size_t
    return int(f(T, B, H, D, V))


@_timed
def delta(proj: torch.Tensor, step: "StepDesc", d: "DeltaDesc", wz: Optional[torch.Tensor], state: torch.Tensor, out: torch.Tensor, scratch: Optional[torch.Tensor] = None):
    """wz f32 [T, H * D]: low-rank branch output (steps with portions; None in steps of single tokens, where the kernel applies w2 itself)"""
    _, _, ld = _rows2d(proj)
    assert out.is_contiguous() and state.is_contiguous() and (scratch is None or (scratch.dtype == torch.float32 and scratch.is_contiguous()))
    _check(lib().b200seq_delta(_p(proj), ld, C.byref(step), C.byref(d), _p(wz), wz.stride(0) if wz is not None else 0, _p(state), _p(out),
                               _DT[out.dtype], _p(scratch), scratch.numel() if scratch is not None else 0, _st(proj)))


def position_frequencies(width: int, base: float) -> torch.Tensor:
    """f32 [2, ceil(width / 2)]: base^(-2i / width) as high and low parts"""
    import numpy as np
    f = base ** (-2.0 * np.arange((width + 1) // 2, dtype=np.float64) / width)
    hi = f.astype(np.float32)
    return torch.from_numpy(np.stack([hi, (f - hi.astype(np.float64)).astype(np.float32)]))


@_timed
def embed_pos(table: torch.Tensor, ids: torch.Tensor, step: "StepDesc", scale: float, freq: Optional[torch.Tensor], x: torch.Tensor, eps: float, *,
              x0: Optional[torch.Tensor] = None, add_vec: Optional[torch.Tensor] = None, fin_w: Optional[torch.Tensor] = None, a: Optional[torch.Tensor] = None):
    """x[t] = table[ids[t]] * scale + sinusoid(pos) (+ add_vec); x0: the same without add_vec; a: x, normed with fin_w when given, in its own type"""
    W = x.shape[-1]
    assert table.dtype == torch.bfloat16 and table.is_contiguous() and x.is_contiguous() and (freq is None or tuple(freq.shape) == (2, (W + 1) // 2))
    _check(lib().b200seq_embed_pos(_p(table), _p(ids), C.byref(step), scale, _p(freq), W, _p(x0), _p(add_vec), _p(x), _p(fin_w), eps, _p(a),
                                   _DT[a.dtype] if a is not None else F32, _st(x)))


@_timed
def sandwich_norm(x: torch.Tensor, eps: float, *, y: Optional[torch.Tensor] = None, w: Optional[torch.Tensor] = None, add_row: Optional[torch.Tensor] = None,
                  add_vec: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None, x_out: Optional[torch.Tensor] = None, a_out: Optional[torch.Tensor] = None,
                  fin_w: Optional[torch.Tensor] = None):
    """n = x + rms_norm(y) * w + add_row + add_vec; x_out = n, a_out = n (normed with fin_w when given); rows: only these token rows (a_out is row-compact)"""
    W = x.shape[-1]
    R = x.shape[0] if rows is None else rows.numel()
    assert x.is_contiguous() and (y is None or y.is_contiguous()) and (a_out is None or a_out.is_contiguous()) and (add_row is None or add_row.is_contiguous())
    _check(lib().b200seq_sandwich_norm(_p(x), _p(y), _p(w), eps, _p(add_row), _p(add_vec), W, _p(rows), R, _p(x_out), _p(a_out),
                                       _DT[a_out.dtype] if a_out is not None else F32, _p(fin_w), _st(x)))


@_timed
def token_gate(z: torch.Tensor, table: torch.Tensor, col: int, ids: torch.Tensor, out: torch.Tensor):
    """out[t] = gelu_tanh(z[t]) * table[ids[t]][col : col + dim]"""
    T, dim, ldz = _rows2d(z)
    assert table.dtype == torch.bfloat16 and table.is_contiguous() and out.is_contiguous() and tuple(out.shape) == (T, dim)
    _check(lib().b200seq_token_gate(_p(z), ldz, T, dim, _p(table), table.shape[1], col, _p(ids), _p(out), _DT[out.dtype], _st(z)))


@_timed
def side_close(x: torch.Tensor, y: torch.Tensor, w: torch.Tensor, eps: float, gate: torch.Tensor, proj: torch.Tensor, table: torch.Tensor, col: int, ids: torch.Tensor,
               side_w: torch.Tensor, *, add_row: Optional[torch.Tensor] = None, add_vec: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None, x_out: Optional[torch.Tensor] = None,
               a_out: Optional[torch.Tensor] = None, fin_w: Optional[torch.Tensor] = None):
    """sandwich_norm of a sublayer's result, the token-dependent addition and the next norm in one kernel (steps of few tokens; a block per row)"""
    W = x.shape[1]
    R = x.shape[0] if rows is None else rows.numel()
    dim = gate.shape[0]
    assert x.is_contiguous() and y.is_contiguous() and tuple(gate.shape) == (dim, W) and tuple(proj.shape) == (W, dim) and gate.is_contiguous() and proj.is_contiguous()
    assert gate.dtype == proj.dtype == table.dtype == torch.bfloat16 and table.is_contiguous()
    _check(lib().b200seq_side_close(_p(x), _p(y), _p(w), eps, _p(gate), _p(proj), _p(table), table.shape[1], col, dim, _p(ids), _p(side_w),
                                    _p(add_row), _p(add_vec), W, _p(rows), R, _p(x_out), _p(a_out), _DT[a_out.dtype] if a_out is not None else F32, _p(fin_w), _st(x)))


# ---- routing with every constant given; selective scan; residual of parallel layers ------------------------------------------------------------
class RouteDesc(C.Structure):
    """b200seq_route_desc: sizes and constants of a router's choice"""
    _fields_ = [("E", C.c_int32), ("groups", C.c_int32), ("keep", C.c_int32), ("top", C.c_int32), ("kind", C.c_int32), ("group_best", C.c_int32), ("renorm", C.c_int32),
                ("scale", C.c_float), ("correction", C.c_void_p)]


def route_desc(E: int, groups: int, keep: int, top: int, kind: int, *, group_best: int = 2, renorm: bool = True, scale: float = 1.0,
               correction: Optional[torch.Tensor] = None) -> "RouteDesc":
    """group_best: a group's score is the sum of its two largest scores (2) or its largest (1); renorm: weights divided by their sum; the caller keeps correction alive"""
    assert correction is None or (correction.dtype == torch.float32 and correction.numel() == E)
    return RouteDesc(E, groups, keep, top, kind, group_best, int(renorm), scale, correction.data_ptr() if correction is not None else None)


@_timed
def moe_route_rule(z: torch.Tensor, d: "RouteDesc", ids: torch.Tensor, wts: torch.Tensor, counts: Optional[torch.Tensor]):
    T, _, ldz = _rows2d(z)
    assert ids.dtype == torch.int32 and wts.dtype == torch.float32 and ids.is_contiguous() and wts.is_contiguous() and ids.numel() >= T * d.top
    _check(lib().b200seq_moe_route_rule(_p(z), ldz, T, C.byref(d), _p(ids), _p(wts), _p(counts), _st(z)))


@_timed
def moe_router_rule(x: torch.Tensor, w: torch.Tensor, d: "RouteDesc", z: torch.Tensor, ids: torch.Tensor, wts: torch.Tensor):
    """router projection and choice of at most 8 tokens in one kernel"""
    T, K, ldx = _rows2d(x)
    _, NR, ldz = _rows2d(z)
    assert w.dtype == torch.bfloat16 and w.is_contiguous() and tuple(w.shape) == (NR, K) and z.dtype == torch.float32 and z.shape[0] == T
    _check(lib().b200seq_moe_router_rule(_p(x), _DT[x.dtype], ldx, _p(w), T, NR, K, C.byref(d), _p(z), ldz, _p(ids), _p(wts), _st(x)))


class ScanDesc(C.Structure):
    """b200seq_scan_desc: sizes and weights of one selective scan"""
    _fields_ = [("C", C.c_int32), ("N", C.c_int32), ("R", C.c_int32), ("a2", C.c_void_p), ("D", C.c_void_p), ("dt_b", C.c_void_p), ("w_dt", C.c_void_p)]


def scan_desc(a2: torch.Tensor, D: torch.Tensor, dt_b: torch.Tensor, w_dt: torch.Tensor) -> "ScanDesc":
    """a2 f32 [C, N] = A * log2(e); D, dt_b f32 [C]; w_dt bf16 [C, R]; the caller keeps the tensors alive"""
    Cn, N = a2.shape
    assert a2.dtype == D.dtype == dt_b.dtype == torch.float32 and w_dt.dtype == torch.bfloat16 and D.numel() == dt_b.numel() == w_dt.shape[0] == Cn
    assert a2.is_contiguous() and D.is_contiguous() and dt_b.is_contiguous() and w_dt.is_contiguous()
    return ScanDesc(Cn, N, w_dt.shape[1], a2.data_ptr(), D.data_ptr(), dt_b.data_ptr(), w_dt.data_ptr())


def scan_scratch_floats(T: int, B: int, Cn: int, N: int) -> int:
    """floats of work area a selective-scan step of T tokens in B entries wants (0: none)"""
    f = lib().b200seq_scan_scratch_floats
    f.restype = C.c_size_t
    return int(f(T, B, Cn, N))


@_timed
def selective_scan(u: torch.Tensor, dbc: torch.Tensor, dtz: Optional[torch.Tensor], gate: torch.Tensor, step: "StepDesc", d: "ScanDesc", state: torch.Tensor, out: torch.Tensor,
                   scratch: Optional[torch.Tensor] = None):
    """u [T, C]; dbc f32 [T, R + 2 N]; dtz f32 [T, C] (steps with portions; overwritten); gate f32 [T, C] view, already activated; state f32 [slots, C, N]"""
    T, _, ldd = _rows2d(dbc)
    _, _, ldg = _rows2d(gate)
    assert u.is_contiguous() and u.shape[1] == d.C and out.is_contiguous() and out.shape[1] == d.C and state.is_contiguous() and tuple(state.shape[1:]) == (d.C, d.N)
    assert dbc.dtype == gate.dtype == state.dtype == torch.float32 and (dtz is None or (dtz.dtype == torch.float32 and dtz.is_contiguous() and dtz.shape[1] == d.C))
    assert scratch is None or (scratch.dtype == torch.float32 and scratch.is_contiguous())
    _check(lib().b200seq_selective_scan(_p(u), _DT[u.dtype], _p(dbc), ldd, _p(dtz), _p(gate), ldg, C.byref(step), C.byref(d), _p(state), _p(out),
                                        _DT[out.dtype], _p(scratch), scratch.numel() if scratch is not None else 0, _st(dbc)))


class ParallelDesc(C.Structure):
    """b200seq_parallel_desc"""
    _fields_ = [("x", C.c_void_p), ("y1", C.c_void_p), ("w_b1", C.c_void_p), ("ss1", C.c_void_p), ("ss_n", C.c_int32), ("ss_count", C.c_int32), ("s1", C.c_float),
                ("y2", C.c_void_p), ("w_b2", C.c_void_p), ("s2", C.c_float), ("y3", C.c_void_p), ("ys", C.c_void_p), ("wts", C.c_void_p), ("slot_of", C.c_void_p),
                ("top", C.c_int32), ("mult", C.c_float), ("add_vec", C.c_void_p), ("eps", C.c_float), ("W", C.c_int32), ("rows", C.c_void_p), ("R", C.c_int32),
                ("x_out", C.c_void_p), ("a_out", C.c_void_p), ("out_dtype", C.c_int32), ("fin_w", C.c_void_p)]


@_timed
def parallel_close(x: torch.Tensor, y1: torch.Tensor, mult: float, eps: float, *, w_b1: Optional[torch.Tensor] = None, sumsq: Optional[torch.Tensor] = None, sumsq_count: int = 0,
                   s1: float = 1.0, y2: Optional[torch.Tensor] = None, w_b2: Optional[torch.Tensor] = None, s2: float = 1.0, y3: Optional[torch.Tensor] = None,
                   ys: Optional[torch.Tensor] = None, wts: Optional[torch.Tensor] = None, slot_of: Optional[torch.Tensor] = None, top: int = 0,
                   add_vec: Optional[torch.Tensor] = None, rows: Optional[torch.Tensor] = None, x_out: Optional[torch.Tensor] = None, a_out: Optional[torch.Tensor] = None,
                   fin_w: Optional[torch.Tensor] = None):
    """n = x + mult * (s1 b1 + s2 b2 + ff) + add_vec; b1 = y1, rms-normed with w_b1 or divided by the root of its deferred norm (sumsq [T, P], over sumsq_count
    elements); b2 = y2 (rms-normed with w_b2); ff = y3 or the weighted sum of a token's expert rows ys; x_out = n, a_out = n (normed with fin_w when given)"""
    W = x.shape[-1]
    R = x.shape[0] if rows is None else rows.numel()
    assert all(t is None or (t.is_contiguous() and t.dtype == torch.float32) for t in (x, y1, y2, y3, ys, wts, sumsq, x_out, add_vec)) and (a_out is None or a_out.is_contiguous())
    ptr = lambda t: t.data_ptr() if t is not None else None
    d = ParallelDesc(ptr(x), ptr(y1), ptr(w_b1), ptr(sumsq), sumsq.shape[1] if sumsq is not None else 0, sumsq_count, s1, ptr(y2), ptr(w_b2), s2, ptr(y3), ptr(ys), ptr(wts),
                     ptr(slot_of), top, mult, ptr(add_vec), eps, W, ptr(rows), R, ptr(x_out), ptr(a_out), _DT[a_out.dtype] if a_out is not None else F32, ptr(fin_w))
    _check(lib().b200seq_parallel_close(C.byref(d), _st(x)))


# ---- a KV cache held in 4 bits -----------------------------------------------------------------------------------------------------------------------
KV4_MAX_DIM = 128
_U8 = torch.uint8


def kv4_page_bytes(block_size: int, heads: int, dim: int) -> int:
    """bytes of one page of `block_size` positions: 0.625 a value (heads of up to 32, 64 or 128 values are held as that many)"""
    n = int(lib().b200seq_kv4_page_bytes(block_size, heads, dim))
    if n == 0:
        raise ValueError(f"a 4-bit cache holds heads of 1 to {KV4_MAX_DIM} values, not pages of {block_size} positions of {heads} heads of {dim}")
    return n


def kv4_pool(num_blocks: int, block_size: int, heads: int, dim: int, device) -> torch.Tensor:
    """uint8 pool of zeroed pages [num_blocks, heads, bytes of a head's page] for rows of `heads` heads of `dim` values (layout: include/b200seq.h)"""
    return torch.zeros((num_blocks, heads, kv4_page_bytes(block_size, 1, dim)), dtype=torch.uint8, device=device)


def _on_device(name: str, fn, args: tuple, *tensors: Optional[torch.Tensor]) -> None:
    """a library call on the one CUDA device of its tensors, on that device's current stream (the library launches on the current device)"""
    dev = -2
    for t in tensors:
        if t is not None:
            d = t.get_device()
            if d != dev:
                if dev != -2 or d < 0:
                    raise ValueError(f"{name}: tensors of one cuda device expected, but got: {[str(t.device) for t in tensors if t is not None]}")
                dev = d
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc != 0:
        _check(rc)


def _kv4_pool_check(name: str, what: str, pool: torch.Tensor, shape: torch.Size, block_size: int, heads: int, dim: int) -> None:
    if pool.dtype != _U8 or len(shape) != 3 or shape[1] != heads or shape[2] != 20 * block_size * (1 if dim <= 32 else 2 if dim <= 64 else 4) or not pool.is_contiguous():
        raise ValueError(f"{name}: the {what} pool is no contiguous uint8 [pages, {heads}, bytes] of pages of {block_size} positions and heads of {dim} values: "
                         f"{pool.dtype} {tuple(shape)}")


def _kv4_rows(name: str, k: torch.Tensor, v: torch.Tensor, kpool: torch.Tensor, vpool: torch.Tensor, step: "StepDesc"):
    """(heads, size) of keys, the same of values, row strides"""
    ks, vs, kt, vt, T, kp, vp = k.shape, v.shape, k.stride(), v.stride(), step.T, kpool.shape, vpool.shape
    if len(kp) != 3 or len(vp) != 3 or not kp[1] or not vp[1]:
        raise ValueError(f"{name}: pools are uint8 [pages, heads, bytes], not {tuple(kp)} and {tuple(vp)}")
    G, Gv = kp[1], vp[1]
    if len(ks) != 2 or len(vs) != 2 or kt[1] != 1 or vt[1] != 1 or ks[0] != T or vs[0] != T or ks[1] % G or vs[1] % Gv or k.dtype != v.dtype:
        raise ValueError(f"{name}: rows {tuple(ks)} and {tuple(vs)} of {T} tokens do not fit {G} and {Gv} heads")
    D, V, bs = ks[1] // G, vs[1] // Gv, step.block_size
    _kv4_pool_check(name, "key", kpool, kp, bs, G, D)
    _kv4_pool_check(name, "value", vpool, vp, bs, Gv, V)
    return G, D, Gv, V, kt[0], vt[0]


@_timed
def kv4_store(k: torch.Tensor, v: torch.Tensor, step: "StepDesc", kpool: torch.Tensor, vpool: torch.Tensor):
    """keys [T, G * D] and values [T, Gv * V] (f32 or bf16 rows, as they are to be cached: normed, rotated) of the step's tokens go to their pages, quantised to 4 bits"""
    G, D, Gv, V, ldk, ldv = _kv4_rows("kv4_store", k, v, kpool, vpool, step)
    dt = _DT.get(k.dtype)
    if dt is None:
        raise ValueError(f"kv4_store: rows are float32 or bfloat16, not {k.dtype}")
    _on_device("kv4_store", lib().b200seq_kv4_store, (k.data_ptr(), ldk, v.data_ptr(), ldv, dt, C.byref(step), G, D, Gv, V, kpool.data_ptr(), vpool.data_ptr()), k, v, kpool, vpool)


@_timed
def kv4_load(kpool: torch.Tensor, vpool: torch.Tensor, step: "StepDesc", k: torch.Tensor, v: torch.Tensor):
    """the rows that the cache holds for the step's tokens, as the values they stand for: k f32 [T, G * D], v f32 [T, Gv * V]"""
    G, D, Gv, V, ldk, ldv = _kv4_rows("kv4_load", k, v, kpool, vpool, step)
    if k.dtype != torch.float32:
        raise ValueError(f"kv4_load: rows are float32, not {k.dtype}")
    _on_device("kv4_load", lib().b200seq_kv4_load, (kpool.data_ptr(), vpool.data_ptr(), C.byref(step), G, D, Gv, V, k.data_ptr(), ldk, v.data_ptr(), ldv), k, v, kpool, vpool)


def _kv4_layer(name: str, proj: torch.Tensor, step: "StepDesc", d: "AttnDesc", kpool: Optional[torch.Tensor], vpool: Optional[torch.Tensor], need: int) -> int:
    shape, ld = proj.shape, proj.stride()
    if len(shape) != 2 or ld[1] != 1 or proj.dtype != torch.float32 or shape[0] < step.T or shape[1] < need:
        raise ValueError(f"{name}: projection rows are row-major float32 [{step.T}, {need} or more], not {proj.dtype} {tuple(shape)}")
    G, bs = d.G, step.block_size
    if kpool is not None:
        _kv4_pool_check(name, "key", kpool, kpool.shape, bs, G, d.D)
    if vpool is not None:
        _kv4_pool_check(name, "value", vpool, vpool.shape, bs, d.vg if d.vg > 0 else G, d.V)
    return ld[0]


@_timed
def attn_prep_kv4(proj: torch.Tensor, step: "StepDesc", d: "AttnDesc", kpool: Optional[torch.Tensor], vpool: Optional[torch.Tensor], rot_pos: Optional[torch.Tensor] = None):
    """attn_prep_ex over a 4-bit cache: queries biased, normed and rotated in place, keys and values likewise into their pages"""
    if rot_pos is not None:
        d = _turned("attn_prep_kv4", step, d, rot_pos)
    need = max(d.q_col + d.H * d.D, 0 if d.kv_shared else max(d.k_col + d.G * d.D, d.v_col + (d.vg if d.vg > 0 else d.G) * d.V))
    ld = _kv4_layer("attn_prep_kv4", proj, step, d, kpool, vpool, need)
    _on_device("attn_prep_kv4", lib().b200seq_attn_prep_kv4, (_p(proj), ld, C.byref(step), C.byref(d), _p(kpool), _p(vpool)), proj, kpool, vpool)


@_timed
def attn_kv4(proj: torch.Tensor, step: "StepDesc", d: "AttnDesc", kpool: torch.Tensor, vpool: torch.Tensor, out: torch.Tensor, gate: Optional[torch.Tensor] = None,
             max_keys: int = 0):
    """attn_ex over a 4-bit cache: out [T, H * V] (f32 or bf16) = softmax(q k^T * scale + mask) v, gated as the layer says.  max_keys: keys of the step's longest
    sequence, where the block tables hold many more (0: as many as they hold); the work is shared out by it, results do not depend on it but for roundings.
    (The work area of few long sequences is the call's own: no two calls, streams or graphs share it.)"""
    H, V, T = d.H, d.V, step.T
    need = d.q_col + H * d.D
    if d.gate_col >= 0 and gate is None and not d.gate:
        need = max(need, d.gate_col + (H * V if d.gate_elem else H))
    ld = _kv4_layer("attn_kv4", proj, step, d, kpool, vpool, need)
    dt, shape = _DT.get(out.dtype), out.shape
    if dt is None or len(shape) < 2 or shape[0] < T or (shape[1] if len(shape) == 2 else out.numel() // max(1, shape[0])) != H * V or not out.is_contiguous():
        raise ValueError(f"attn_kv4: results are contiguous float32 or bfloat16 [{T}, {H * V}], not {out.dtype} {tuple(shape)}")
    if gate is not None:
        if gate.dim() != 2 or gate.stride(1) != 1 or gate.dtype != torch.float32 or gate.shape[0] < T or gate.shape[1] < (H * V if d.gate_elem else H):
            raise ValueError("attn_kv4: gate logits are row-major float32 rows, one for each head (or output element)")
        d2 = AttnDesc.from_buffer_copy(d)
        d2.gate, d2.gate_ld = gate.data_ptr(), gate.stride(0)
        d = d2
    L = lib()
    sref, dref = C.byref(step), C.byref(d)
    need = L.b200seq_attn_kv4_scratch_floats(sref, dref, max_keys)
    scratch = torch.empty(need, dtype=torch.float32, device=proj.device) if need else None
    _on_device("attn_kv4", L.b200seq_attn_kv4, (proj.data_ptr(), ld, sref, dref, kpool.data_ptr(), vpool.data_ptr(), out.data_ptr(), dt, scratch.data_ptr() if need else None, need, max_keys),
               proj, kpool, vpool, out, gate)


# ---- pages ---------------------------------------------------------------------------------------------------------------------------------------------
@_timed
def copy_pages(pools: Sequence[torch.Tensor], pairs: Sequence[Tuple[int, int]]):
    """page `to` of every pool <- its page `from`, for all pairs (from, to) of host numbers, in one launch.  Pools: contiguous, the first dimension counts the
    pages and is the same in all.  A page may be read by several pairs, but not written twice and not both read and written."""
    n = len(pairs)
    if not len(pools):
        return
    pages = pools[0].shape[0]
    ptrs, size = [], []
    for p in pools:
        if p.shape[0] != pages or not p.is_contiguous():
            raise ValueError(f"copy_pages: pools are contiguous and of one number of pages, not {tuple(p.shape)} beside {pages}")
        ptrs.append(p.data_ptr())
        size.append(p.nbytes // pages if pages else 0)
    try:
        flat = pack(f"{2 * n}i", *chain.from_iterable(pairs))
    except StructError as e:
        raise ValueError(f"copy_pages: pairs of (from, to) numbers expected: {e}") from None
    np_ = len(ptrs)
    _on_device("copy_pages", lib().b200seq_copy_pages, (pack(f"{np_}P", *ptrs), pack(f"{np_}q", *size), np_, pages, flat, n), *pools)


# ---- sampling rules ------------------------------------------------------------------------------------------------------------------------------------
@_timed
def process_logits(logits: torch.Tensor, rules: torch.Tensor, out: Optional[torch.Tensor] = None, *, hist: Optional[torch.Tensor] = None, hist_start: Optional[torch.Tensor] = None,
                   hist_prompt: Optional[torch.Tensor] = None, bias_start: Optional[torch.Tensor] = None, bias_ids: Optional[torch.Tensor] = None,
                   bias_vals: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out [R, V] f32 (default: `logits` in place): penalties for the tokens of each row's history, biases, temperature and a mask (include/b200seq.h has the order).
    rules f32 [R, 4]: repetition, presence, frequency, temperature.  hist int32 [total] with hist_start int32 [R + 1] and hist_prompt int32 [R] (how many of a
    row's ids are its prompt); bias_ids int32, bias_vals f32 with bias_start int32 [R + 1]; mask int32 [R, ceil(V / 32)], bit v % 32 of word v / 32 set: allowed."""
    out = logits if out is None else out
    shape, lx, lo = logits.shape, logits.stride(), out.stride()
    if len(shape) != 2 or out.shape != shape or lx[1] != 1 or lo[1] != 1 or logits.dtype != torch.float32 or out.dtype != torch.float32:
        raise ValueError(f"process_logits: row-major float32 logits and results of one shape, not {logits.dtype} {tuple(shape)} and {out.dtype} {tuple(out.shape)}")
    R, V = shape
    words = (V + 31) // 32
    i32, f32 = torch.int32, torch.float32
    for name, t, dtype, n in (("rules", rules, f32, 4 * R), ("hist", hist, i32, None), ("hist_start", hist_start, i32, R + 1), ("hist_prompt", hist_prompt, i32, R),
                              ("bias_start", bias_start, i32, R + 1), ("bias_ids", bias_ids, i32, None), ("bias_vals", bias_vals, f32, bias_ids.numel() if bias_ids is not None else None)):
        if t is not None and (t.dtype != dtype or not t.is_contiguous() or (n is not None and t.numel() != n)):
            raise ValueError(f"process_logits: {name} is contiguous {dtype}{'' if n is None else f' of {n} values'}, not {t.dtype} {tuple(t.shape)}")
    lm = 0
    if mask is not None:
        lm = mask.stride()
        if len(lm) != 2 or lm[1] != 1 or mask.dtype != i32 or mask.shape[0] != R or mask.shape[1] < words:
            raise ValueError(f"process_logits: the mask is row-major int32 [{R}, {words}], not {mask.dtype} {tuple(mask.shape)}")
        lm = max(lm[0], words) if R == 1 else lm[0]
    if hist is not None and hist.numel() == 0:      # histories without a token
        hist = hist_start = hist_prompt = None
    if bias_ids is not None and bias_ids.numel() == 0:
        bias_ids = bias_start = bias_vals = None
    _on_device("process_logits", lib().b200seq_process_logits,
               (logits.data_ptr(), lx[0] if R > 1 else V, R, V, rules.data_ptr(), _p(hist), hist.numel() if hist is not None else 0, _p(hist_start), _p(hist_prompt),
                _p(bias_start), _p(bias_ids), _p(bias_vals), bias_ids.numel() if bias_ids is not None else 0, _p(mask), lm, out.data_ptr(), lo[0] if R > 1 else V), logits, rules, out, hist, hist_start, hist_prompt, bias_start, bias_ids, bias_vals, mask)
    return out


# ---- drafts, and a cache of bounded size -----------------------------------------------------------------------------------------------------------------
def _flat(name: str, what: str, t: Optional[torch.Tensor], dtype, n: int) -> None:
    if t is not None and (t.dtype != dtype or t.numel() != n or not t.is_contiguous()):
        raise ValueError(f"{name}: {what} is contiguous {dtype} of {n} values, not {t.dtype} {tuple(t.shape)}")


@_timed
def verify_drafts(logits: torch.Tensor, start: torch.Tensor, drafts: torch.Tensor, accept_u: torch.Tensor, sample_u: torch.Tensor, temperature: torch.Tensor, *,
                  top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None, draft_probs: Optional[torch.Tensor] = None,
                  accepted: Optional[torch.Tensor] = None, tokens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """drafted tokens against the probabilities of f32 logits [R, V], from given random numbers.  Entry e has rows start[e] .. start[e + 1] - 1 (start int32 [B + 1]): its drafts
    (drafts int32 [R], one a row) and one row more; an entry of one row samples a token.  A draft x is accepted when accept_u * q(x) < p(x) (accept_u f32 [R], draft_probs f32 [R, V]
    the distributions it was drawn from; None: it was certain); the token behind the accepted ones is drawn with sample_u (f32 [B]) from what p has more than q, or from the last
    row's p.  temperature f32 [B] (0: the largest logit, always), top_k int32 [B] (0: all), top_p f32 [B] (1: all) make p as include/b200seq.h says.
    Returns (accepted int32 [B], tokens int32 [R]: accepted drafts, the token behind them, then -1; -1 in its place: the row's logits leave no choice)."""
    shape, lx = logits.shape, logits.stride()
    if len(shape) != 2 or lx[1] != 1 or logits.dtype != torch.float32 or shape[1] < 1:
        raise ValueError(f"verify_drafts: row-major float32 logits [rows, vocabulary], not {logits.dtype} {tuple(shape)}")
    R, V = shape
    B = temperature.numel()
    i32, f32 = torch.int32, torch.float32
    accepted = torch.empty(B, dtype=i32, device=logits.device) if accepted is None else accepted
    tokens = torch.empty(R, dtype=i32, device=logits.device) if tokens is None else tokens
    for what, t, dtype, n in (("start", start, i32, B + 1), ("drafts", drafts, i32, R), ("accept_u", accept_u, f32, R), ("sample_u", sample_u, f32, B), ("temperature", temperature, f32, B),
                              ("top_k", top_k, i32, B), ("top_p", top_p, f32, B), ("accepted", accepted, i32, B), ("tokens", tokens, i32, R)):
        _flat("verify_drafts", what, t, dtype, n)
    lq = 0
    if draft_probs is not None:
        lq = draft_probs.stride()
        if draft_probs.shape != shape or lq[1] != 1 or draft_probs.dtype != f32:
            raise ValueError(f"verify_drafts: draft_probs are row-major float32 {tuple(shape)}, not {draft_probs.dtype} {tuple(draft_probs.shape)}")
        lq = lq[0] if R > 1 else V
    L = lib()
    need = L.b200seq_verify_scratch_bytes(R, V, top_k is not None or top_p is not None)
    scratch = torch.empty(need, dtype=_U8, device=logits.device)
    _on_device("verify_drafts", L.b200seq_verify_drafts,
               (logits.data_ptr(), lx[0] if R > 1 else V, R, V, start.data_ptr(), B, drafts.data_ptr(), accept_u.data_ptr(), sample_u.data_ptr(), temperature.data_ptr(), _p(top_k),
                _p(top_p), _p(draft_probs), lq, accepted.data_ptr(), tokens.data_ptr(), scratch.data_ptr(), need),
               logits, start, drafts, accept_u, sample_u, temperature, top_k, top_p, draft_probs, accepted, tokens)
    return accepted, tokens


@_timed
def key_weights(proj: torch.Tensor, step: "StepDesc", d: "AttnDesc", kpool: torch.Tensor, acc: torch.Tensor, *, last: int = 0, max_keys: int = 0):
    """adds up the soft-max weight that the step's tokens (their queries prepared in proj) give to the cached keys of their sequences: acc f32 [slots, G, room], by the entries' state
    slots; keys that the step brought begin at zero.  kpool: the layer's f32 or 4-bit key pages.  last: only that many last tokens of every entry count (0: all).  max_keys: keys of the
    step's longest sequence, where the block tables hold many more (0: as many as they hold; never fewer than it has)."""
    four = kpool.dtype == _U8
    shape, ld = proj.shape, proj.stride()
    if len(shape) != 2 or ld[1] != 1 or proj.dtype != torch.float32 or shape[0] < step.T or shape[1] < d.q_col + d.H * d.D:
        raise ValueError(f"key_weights: projection rows are row-major float32 [{step.T}, {d.q_col + d.H * d.D} or more], not {proj.dtype} {tuple(shape)}")
    if four:
        _kv4_pool_check("key_weights", "key", kpool, kpool.shape, step.block_size, d.G, d.D)
    elif kpool.dtype != torch.float32 or kpool.dim() != 4 or tuple(kpool.shape[1:]) != (step.block_size, d.G, d.D) or not kpool.is_contiguous():
        raise ValueError(f"key_weights: the key pool is contiguous float32 [pages, {step.block_size}, {d.G}, {d.D}], not {kpool.dtype} {tuple(kpool.shape)}")
    if acc.dtype != torch.float32 or acc.dim() != 3 or acc.shape[1] != d.G or not acc.is_contiguous() or acc.numel() == 0:
        raise ValueError(f"key_weights: weights are contiguous float32 [slots, {d.G}, room], not {acc.dtype} {tuple(acc.shape)}")
    if last < 0 or max_keys < 0:
        raise ValueError(f"key_weights: last {last} tokens of {max_keys} keys")
    L = lib()
    sref, dref = C.byref(step), C.byref(d)
    need = L.b200seq_key_weights_scratch_floats(sref, dref, last, max_keys)
    scratch = torch.empty(max(need, 4), dtype=torch.float32, device=proj.device)
    _on_device("key_weights", L.b200seq_key_weights, (proj.data_ptr(), ld[0], sref, dref, kpool.data_ptr(), 4 if four else 32, acc.data_ptr(), acc.shape[0], acc.shape[2], last, max_keys,
                                                      scratch.data_ptr(), need), proj, kpool, acc)


@_timed
def evict_keys(kpools: Sequence[torch.Tensor], vpools: Sequence[torch.Tensor], accs: Sequence[torch.Tensor], slots: torch.Tensor, rows: torch.Tensor, table: torch.Tensor, keep: int, *,
               first: int = 0, recent: int = 0, block_size: int = 0, to_table: Optional[torch.Tensor] = None, to_slots: Optional[torch.Tensor] = None,
               kept: Optional[torch.Tensor] = None) -> torch.Tensor:
    """sequences of more than `keep` cached rows are cut back, in every layer and key head for itself, to the `first` ones, the `recent` ones and those of largest weight between: rows of
    keys, values and weights go, in order, to the places 0 .. keep - 1 of to_table and to_slots (default: where they are).  Layers: lists of pools (f32 [pages, block_size, G, D] or
    4-bit ones, for which block_size is given) and of their weights f32 [slots, G, room]; entries: slots int32 [B], rows int32 [B] (how many each has), table int32 [B, pages].
    No two entries write into one page or slot.  Returns kept int32 [layers, B, G, keep]: the rows that stayed, -1 behind them."""
    n, i32 = len(kpools), torch.int32
    if n == 0 or len(vpools) != n or len(accs) != n:
        raise ValueError(f"evict_keys: {n} key pools, {len(vpools)} value pools and {len(accs)} weights")
    k, v, a = kpools[0], vpools[0], accs[0]
    four = k.dtype == _U8
    if four:
        if block_size < 1:
            raise ValueError("evict_keys: 4-bit pools need their block size")
        if k.dim() != 3 or v.dim() != 3 or any(p.shape[2] not in (20 * block_size, 40 * block_size, 80 * block_size) for p in (k, v)):
            raise ValueError(f"evict_keys: pools {tuple(k.shape)} and {tuple(v.shape)} are not of pages of {block_size} positions")
        bs, G, Gv = block_size, k.shape[1], v.shape[1]
        D, V = (p.shape[2] // (20 * bs) * 32 for p in (k, v))
    else:
        if k.dim() != 4 or v.dim() != 4 or k.shape[1] != v.shape[1] or block_size not in (0, k.shape[1]):
            raise ValueError(f"evict_keys: pools {tuple(k.shape)} and {tuple(v.shape)} are not of one block size")
        bs, G, D, Gv, V = k.shape[1], k.shape[2], k.shape[3], v.shape[2], v.shape[3]
    for what, ts, like, dtype in (("key pools", kpools, k, k.dtype if four else torch.float32), ("value pools", vpools, v, k.dtype if four else torch.float32), ("weights", accs, a, torch.float32)):
        for t in ts:
            if t.dtype != dtype or t.shape != like.shape or not t.is_contiguous():
                raise ValueError(f"evict_keys: {what} are contiguous {dtype} of one shape, not {t.dtype} {tuple(t.shape)} beside {tuple(like.shape)}")
    if k.shape[0] != v.shape[0] or a.dim() != 3 or a.shape[1] != G or a.numel() == 0 or k.numel() == 0 or v.numel() == 0:
        raise ValueError(f"evict_keys: pools {tuple(k.shape)} and {tuple(v.shape)} with weights {tuple(a.shape)}")
    if not (keep >= 1 and first >= 0 and recent >= 0 and first + recent <= keep):
        raise ValueError(f"evict_keys: the first {first} and the last {recent} of {keep} rows to keep")
    B = rows.numel()
    to_table, to_slots = table if to_table is None else to_table, slots if to_slots is None else to_slots
    kept = torch.empty((n, B, G, keep), dtype=i32, device=k.device) if kept is None else kept
    for what, t, m in (("slots", slots, B), ("rows", rows, B), ("to_slots", to_slots, B), ("kept", kept, n * B * G * keep)):
        _flat("evict_keys", what, t, i32, m)
    for what, t in (("table", table), ("to_table", to_table)):
        if t.dtype != i32 or t.dim() != 2 or t.shape[0] != B or t.shape[1] < 1 or not t.is_contiguous():
            raise ValueError(f"evict_keys: {what} is contiguous int32 [{B}, pages], not {t.dtype} {tuple(t.shape)}")
    ptrs = lambda ts: pack(f"{n}P", *[t.data_ptr() for t in ts])
    _on_device("evict_keys", lib().b200seq_evict_keys,
               (ptrs(kpools), ptrs(vpools), ptrs(accs), n, 4 if four else 32, bs, G, D, Gv, V, a.shape[0], a.shape[2], slots.data_ptr(), rows.data_ptr(), table.data_ptr(), table.shape[1],
                to_slots.data_ptr(), to_table.data_ptr(), to_table.shape[1], B, keep, first, recent, kept.data_ptr()), *kpools, *vpools, *accs, slots, rows, table, to_slots, to_table, kept)
    return kept
