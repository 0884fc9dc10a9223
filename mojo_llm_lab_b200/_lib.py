"""ctypes binding of lib/libmllb200.so (the C ABI of include/mllb200.h).

Loading fails loudly: there is no CPU or eager-PyTorch fallback anywhere in
this package.  If the library is missing it is built in place with nvcc; if
that fails the import error propagates.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import re
import threading
from pathlib import Path

from . import build as _build

HEADER = _build.INCLUDE / "mllb200.h"

MLLB_OK = 0
MLLB_EINVAL = -1
MLLB_EALIGN = -2
MLLB_ECUDA = -3
MLLB_EUNSUPPORTED = -4

TYPE_F32 = 0
TYPE_F16 = 1
TYPE_BF16 = 2

LAUNCH_PDL = 1
LAUNCH_CONST_AUX = 2  # IMROPE: gamma / positions / theta not written by the preceding kernel

S_D_SUMQ = 0
S_SUM_X = 1

_P = C.c_void_p
_I64 = C.c_int64


class ActF32(C.Structure):
    """mllb_act_f32 of include/mllb200.h (an activation built in the kernel)."""
    _fields_ = [("x", C.c_void_p), ("delta", C.c_void_p), ("gamma", C.c_void_p), ("x_out", C.c_void_p),
                ("eps", C.c_double), ("advance", C.c_void_p)]


_ACT = C.POINTER(ActF32)



class PeerGather(C.Structure):
    """mllb_peer_gather of include/mllb200.h."""
    _fields_ = [("rank", C.c_int32), ("world", C.c_int32), ("buffers", C.c_void_p * 8),
                ("flags", C.c_void_p * 8), ("count", C.c_void_p)]


class PagedCache(C.Structure):
    """mllb_paged_cache of include/mllb200.h."""
    _fields_ = [("k", _P), ("v", _P), ("pages", _I64), ("kv_heads", _I64), ("page_size", _I64), ("head_dim", _I64),
                ("page_stride", _I64), ("head_stride", _I64), ("row_stride", _I64), ("layers", _I64),
                ("layer_stride", _I64), ("type", C.c_int32)]


class PagedAppend(C.Structure):
    """mllb_paged_append of include/mllb200.h."""
    _fields_ = [("qkv", _P), ("tokens", _I64), ("qkv_stride", _I64), ("positions", _P), ("rows", _P), ("seq", _P),
                ("page_table", _P), ("seqs", _I64), ("table_width", _I64), ("q_gamma", _P), ("k_gamma", _P),
                ("freqs", _P), ("rot_dim", _I64), ("q_heads", _I64), ("eps", C.c_double), ("magnitude", C.c_double),
                ("q_out", _P), ("qkv_type", C.c_int32), ("interleaved", C.c_int32)]


class PagedAttn(C.Structure):
    """mllb_paged_attn of include/mllb200.h."""
    _fields_ = [("q", _P), ("out", _P), ("tokens", _I64), ("q_heads", _I64), ("q_token_stride", _I64),
                ("q_head_stride", _I64), ("out_token_stride", _I64), ("out_head_stride", _I64), ("page_table", _P),
                ("seq_lens", _P), ("seqs", _I64), ("table_width", _I64), ("prefix_table", _P), ("prefix_lens", _P),
                ("group_start", _P), ("groups", _I64), ("prefix_width", _I64), ("q_start", _P), ("scale", C.c_double)]


class BeamScores(C.Structure):
    """mllb_beam_scores of include/mllb200.h."""
    _fields_ = [("logits", _P), ("batch", _I64), ("beams", _I64), ("vocab", _I64), ("n", _I64), ("batch_stride", _I64),
                ("beam_stride", _I64), ("scores", _P), ("done", _P), ("end_token", _I64), ("type", C.c_int32)]


class BeamRows(C.Structure):
    """mllb_beam_rows of include/mllb200.h."""
    _fields_ = [("parents", _P), ("page_table", _P), ("seq_lens", _P), ("fresh", _P), ("batch", _I64), ("beams", _I64),
                ("table_width", _I64)]


SIGNATURES = {
    "mllb_abi_version": (C.c_int, []),
    "mllb_last_error": (C.c_char_p, []),
    "mllb_device_error": (C.c_int, [C.POINTER(C.c_uint32), C.c_int]),
    "mllb_q8_1_quantize": (C.c_int, [_P, _P, _I64, C.c_int, _P]),
    "mllb_q4k_matvec": (C.c_int, [_P, _P, _P, _I64, _I64, _P]),
    "mllb_q4k_matvec_ex": (C.c_int, [_P, _P, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q4k_gate_up_ex": (C.c_int, [_P, _P, _P, _P, _P, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q6k_matvec_ex": (C.c_int, [_P, _P, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q4k_gate_up": (C.c_int, [_P, _P, _P, _P, _P, _P, _I64, _I64, _P]),
    "mllb_q6k_matvec": (C.c_int, [_P, _P, _P, _I64, _I64, _P]),
    "mllb_rmsnorm_imrope_q": (C.c_int, [_P, _P, _P, _P, _P, _I64, _P]),
    "mllb_rmsnorm_imrope_q_batched": (C.c_int, [_P, _P, _P, _P, C.c_double, _P, _I64, _I64, _P]),
    "mllb_rmsnorm_imrope_q_batched_ex": (C.c_int, [_P, _P, _P, _P, C.c_double, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q4k_subdots": (C.c_int, [_P, _P, _P, _P, _I64, _I64, _P]),
    "mllb_stream_read": (C.c_int, [_P, _I64, _P, _I64, _P]),
    "mllb_q8_1_quantize_ex": (C.c_int, [_P, _P, _I64, C.c_int, C.c_uint, _P]),
    "mllb_token_key": (_I64, [C.c_int32]),
    "mllb_key_token": (_I64, [_I64]),
    "mllb_decode_embed": (C.c_int, [_P, _I64, _I64, _P, _P, _I64, _P, C.c_uint, _P]),
    "mllb_rmsnorm_q8_1": (C.c_int, [_P, _P, _P, _P, C.c_double, _P, _I64, C.c_int, C.c_uint, _P]),
    "mllb_decode_final_norm": (C.c_int, [_P, _P, _P, _P, C.c_double, _P, _I64, _P, C.c_uint, _P]),
    "mllb_decode_qk_rope_append": (C.c_int, [_P, _P, _P, _P, C.c_double, _P, _P, _P, _I64, _I64, _I64, C.c_uint,
                                             _P]),
    "mllb_decode_attention_scratch": (_I64, [_I64, _I64, _I64]),
    "mllb_decode_attention": (C.c_int, [_P, _P, _P, _P, _P, _I64, _P, _P, _I64, _I64, _I64, C.c_uint, _P]),
    "mllb_decode_attention_qkv": (C.c_int, [_P, _P, _P, C.c_double, _P, _P, _P, _P, _I64, _P, _P, _I64, _I64, _I64,
                                            C.c_uint, _P]),
    "mllb_decode_attention_qkv_noalloc": (C.c_int, [_P, _P, _P, C.c_double, _P, _P, _P, _P, _P, _I64, _I64, _I64,
                                                    C.c_uint, _P]),
    "mllb_kv_q4_0_store": (C.c_int, [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, C.c_uint, _P]),
    "mllb_decode_attention_q4_0": (C.c_int, [_P, _P, _P, _P, _P, _P, _I64, _P, _P, _I64, _I64, _I64, C.c_uint, _P]),
    "mllb_decode_attention_qkv_q4_0": (C.c_int, [_P, _P, _P, C.c_double, _P, _P, _P, _P, _P, _I64, _P, _P, _I64,
                                                 _I64, _I64, C.c_uint, _P]),
    "mllb_argmax_f32": (C.c_int, [_P, _I64, _I64, _P, C.c_uint, _P]),
    "mllb_q8_1_quantize_allgather": (C.c_int, [_P, _I64, C.POINTER(PeerGather), C.c_uint, _P]),
    "mllb_q4k_gate_up_q8_gather": (C.c_int, [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, C.POINTER(PeerGather),
                                             C.c_uint, _P]),
    "mllb_prefetch_l2": (C.c_int, [_P, _I64, _P]),
    "mllb_q5k_matvec": (C.c_int, [_P, _P, _P, _I64, _I64, _P]),
    "mllb_q5k_matvec_ex": (C.c_int, [_P, _P, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q4k_matvec_act": (C.c_int, [_P, _ACT, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q4k_gate_up_act": (C.c_int, [_P, _P, _ACT, _P, _P, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q6k_matvec_act": (C.c_int, [_P, _ACT, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q4k_gate_up_q8": (C.c_int, [_P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, C.c_uint, _P]),
    "mllb_q4k_matvec_norm_workspace": (_I64, [_I64, _I64]),
    "mllb_q4k_matvec_norm": (C.c_int, [_P, _P, _P, _I64, _I64, _P, _P, _P, C.c_double, _P, _P, _I64, C.c_uint, _P]),
    "mllb_q4k_matmul_tokens_workspace": (C.c_int64, [_I64, _I64, _I64]),
    "mllb_q4k_matmul_tokens": (C.c_int, [_P, _P, _P, _I64, _I64, _I64, _P, _I64, C.c_uint, _P]),
    "mllb_paged_qkv_append": (C.c_int, [C.POINTER(PagedAppend), C.POINTER(PagedCache), C.c_uint, _P]),
    "mllb_paged_attention_workspace": (_I64, [_I64, _I64, _I64, _I64, _I64, _I64]),
    "mllb_paged_attention_call_workspace": (_I64, [C.POINTER(PagedAttn), C.POINTER(PagedCache)]),
    "mllb_paged_attention": (C.c_int, [C.POINTER(PagedAttn), C.POINTER(PagedCache), _P, _I64, C.c_uint, _P]),
    "mllb_beam_select_workspace": (_I64, [_I64, _I64, _I64, _I64]),
    "mllb_beam_select": (C.c_int, [C.POINTER(BeamScores), _P, _P, _P, _P, _I64, C.c_uint, _P]),
    "mllb_beam_reorder": (C.c_int, [C.POINTER(BeamRows), C.POINTER(PagedCache), _P, _P, _P, C.c_uint, _P]),
}

_lock = threading.Lock()
_handle = None
_native = None


class MllbError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"{message} (code {code})")
        self.code = code


def declared_symbols() -> list[str]:
    """Every function the public header declares."""
    text = HEADER.read_text()
    return sorted(set(re.findall(r"^\s*(?:const\s+)?\w+\s*\*?\s*(mllb_\w+)\s*\(", text, re.M)))


def lib() -> C.CDLL:
    global _handle
    with _lock:
        if _handle is None:
            if not _build.LIB.exists():
                _build.build()
            handle = C.CDLL(str(_build.LIB))
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(handle, name)
                fn.restype = res
                fn.argtypes = args
            if handle.mllb_abi_version() != 1:
                raise RuntimeError("libmllb200.so ABI version mismatch")
            _handle = handle
    return _handle


def native():
    """The extension module lib/mllb200_torch.so (csrc/torch_ops.cpp)."""
    global _native
    if _native is None:
        import torch  # noqa: F401  (its libraries are what the extension links to)
        lib()
        with _lock:
            if _native is None:
                if not _build.torch_ext_current():
                    _build.build()
                spec = importlib.util.spec_from_file_location("mllb200_torch", _build.TORCH_EXT)
                module = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(module)
                module.set_error(MllbError)
                _native = module
    return _native


def check(rc: int, what: str) -> None:
    if rc != MLLB_OK:
        msg = lib().mllb_last_error().decode(errors="replace")
        if rc in (MLLB_EINVAL, MLLB_EALIGN):
            raise ValueError(f"{what}: {msg} (code {rc})")
        raise MllbError(rc, f"{what}: {msg}")


def device_error(clear: bool = True) -> int:
    bits = C.c_uint32(0)
    check(lib().mllb_device_error(C.byref(bits), 1 if clear else 0), "mllb_device_error")
    return bits.value
