"""Python host side of the MI355X decode backend: ctypes bindings over the C ABI (include/gemvq_hip.h,
include/gemvq_synth.h) and builders for the command-list words.

The command words mirror the reference kernel's command list (fpga/src/gemvqc16.h:24-135); `Context.run` returns
the same status convention as gemvqc16 (0, the 1-based index of the first invalid command, or a negative error).
The GPU path has no fallback: without the built libgemvq_hip.so or a HIP device, loading fails loudly.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

import numpy as np

PKG = os.path.dirname(os.path.abspath(__file__))
HIP_LIB_PATH = os.path.join(PKG, "libgemvq_hip.so")
SYNTH_LIB_PATH = os.path.join(PKG, "libgemvq_synth.so")

# ggml type ids
Q4_0, Q4_1, Q8_0, Q5_K, Q6_K = 2, 3, 8, 13, 14
# opcodes (gemvqc16.h:100-111 plus the opcodes of this backend)
OP_GEMV, OP_RMSNORM, OP_ADD, OP_SILU_MUL, OP_MUL, OP_UNARY, OP_GDN, OP_CONV, OP_STATE_LOAD, OP_ROPE, OP_TRACE = range(1, 12)
OP_ATTN, OP_GET_ROWS, OP_ARGMAX, OP_NEXT_TOKEN, OP_FILL, OP_GEMM = 12, 13, 14, 15, 16, 17
OP_BEAM, OP_BEAM_MOVE, OP_BEAM_NEXT = 18, 19, 20
BEAM_ACT, BEAM_STATE, BEAM_KV = 0, 1, 2
KV_F16, KV_Q4_0 = 1, 2
ROPE_HALF, ROPE_PAIRS = 0, 1
GEMM_MAX_TOK = 32
GEMV_SWIGLU, GEMV_CONV, GEMV_ADD, GEMV_ARGMAX, GEMV_SILU = 0x100, 0x200, 0x400, 0x800, 0x1000
GDN_WITH_GEMV, GDN_L2_QK, GDN_GATED, GDN_GATES, GDN_WITH_OUT, GDN_Z_SILU, GDN_SEQS = 1, 2, 4, 8, 16, 32, 64
NORM_L2, NORM_NO_WEIGHT, NORM_DEFER = 1, 2, 4
SILU_MUL_SIGMOID = 1
UNARY_SILU, UNARY_SIGMOID, UNARY_SOFTPLUS, UNARY_COPY = 1, 2, 3, 4
EINVAL, ETIMEDOUT, EUNUSABLE = -10000, -10001, -10002
ARITH_CANONICAL, ARITH_REFERENCE = 0, 1
MAX_CMDS = 4096


def fbits(x: float) -> int:
    return struct.unpack("<I", struct.pack("<f", float(x)))[0]


def row_bytes(t: int, cols: int) -> int:
    return {Q4_0: cols // 32 * 18, Q4_1: cols // 32 * 20, Q8_0: cols // 32 * 34, Q5_K: cols // 256 * 176,
            Q6_K: cols // 256 * 210}[t]


# ---------------------------------------------------------------------------------------------------------------
# command builders (8 words each)
def cmd(*words: int) -> list[int]:
    w = [int(x) & 0xFFFFFFFF for x in words]
    assert len(w) <= 8
    return w + [0] * (8 - len(w))


def gemv(fmt: int, rows: int, cols: int, w_off: int, x_off: int, y_off: int, flags: int = 0) -> list[int]:
    return cmd(OP_GEMV, fmt | flags, rows, cols, w_off & 0xFFFFFFFF, w_off >> 32, x_off, y_off)


def rmsnorm(n: int, x_off: int, w_off: int, y_off: int, eps: float, rows: int = 1, flags: int = 0,
            stride_words: int = 0) -> list[int]:
    return cmd(OP_RMSNORM, n, x_off, w_off, y_off, fbits(eps), rows, flags | (stride_words << 8))


def add(n: int, a: int, b: int, y: int) -> list[int]:
    return cmd(OP_ADD, n, a, b, y)


def mul(n: int, a: int, b: int, y: int) -> list[int]:
    return cmd(OP_MUL, n, a, b, y)


def silu_mul(n: int, g: int, u: int, y: int, sigmoid: bool = False, row: int = 0, stride: int = 0) -> list[int]:
    return cmd(OP_SILU_MUL, n, g, u, y, SILU_MUL_SIGMOID if sigmoid else 0, row, stride)


def unary(n: int, x: int, kind: int, y: int, row: int = 0, stride: int = 0) -> list[int]:
    return cmd(OP_UNARY, n, x, kind, y, row, stride)


def conv(ch: int, x: int, w: int, y: int, s_src: int, s_dst: int, silu: bool = True) -> list[int]:
    return cmd(OP_CONV, ch, x, w, y, s_src, s_dst, 1 if silu else 0)


def rope(n_dims: int, x: int, cs: int, y: int, ne0: int, rows: int, pos_off: int = 0) -> list[int]:
    return cmd(OP_ROPE, n_dims, x, cs, y, ne0, rows, pos_off)


def gdn(hv: int, hk: int, q: int, k: int, v: int, g: int, beta: int, y: int, src_row: int, dst_row: int,
        scale: float, flags: int = 0, l2_eps: float = 1e-6, rms_eps: float = 1e-6, w: int = 0, z: int = 0,
        dt: int = 0, a: int = 0) -> list[int]:
    out = cmd(OP_GDN, hv | (hk << 16), q, k, v, g, beta, y)
    out += cmd(src_row, dst_row, fbits(scale), flags, fbits(l2_eps), fbits(rms_eps), w, z)
    if flags & GDN_GATES:
        out += cmd(dt, a)
    return out


def attn(n_head: int, n_head_kv: int, q: int, kv: int, y: int, head_dim: int, n_rot: int, pos_off: int,
         k: int, v: int, scale: float, eps: float, qn: int, kn: int, cs: int, gate: int | None = None,
         n_tok: int = 1) -> list[int]:
    """n_tok > 1: tokens at positions act[pos_off] + t with packed rows (q / gate, k, v and y of token t follow
    those of token t - 1)."""
    flags = (1 if gate is not None else 0) | ((n_tok << 16) if n_tok > 1 else 0)
    out = cmd(OP_ATTN, n_head | (n_head_kv << 16), q, kv, y, head_dim | (n_rot << 16), pos_off, flags)
    out += cmd(k, v, fbits(scale), fbits(eps), qn, kn, cs, gate or 0)
    return out


def get_rows(fmt: int, rows: int, cols: int, w_off: int, id_off: int, y_off: int, n_tok: int = 1) -> list[int]:
    """n_tok > 1: token t's id at act[id_off + 16 t], its row at y_off + t * cols."""
    return cmd(OP_GET_ROWS, fmt | ((n_tok << 16) if n_tok > 1 else 0), rows, cols, w_off & 0xFFFFFFFF, w_off >> 32,
               id_off, y_off)


def argmax(n: int, x: int, key: int) -> list[int]:
    return cmd(OP_ARGMAX, n, x, key)


def next_token(key: int, tok: int, pos: int, prompt: int, n_prompt: int, out: int) -> list[int]:
    return cmd(OP_NEXT_TOKEN, key, tok, pos, prompt, n_prompt, out)


def beam(n_vocab: int, x: int, row_stride: int, n_beam: int, n_group: int, eos: int, score: int, parent: int, tok: int,
         pos: int = 0, plen: int = 0, prompt: int = 0, cap: int = 0) -> list[int]:
    """One step of a beam search over n_group groups of n_beam sequences; slots 16 floats apart."""
    return cmd(OP_BEAM, n_vocab, x, row_stride, n_beam | (n_group << 8), eos, score, parent) + cmd(tok, pos, plen, prompt, cap)


def beam_move(kind: int, off: int, row_stride: int, n: int, parent: int, n_beam: int, n_group: int, n_part: int = 1,
              part_stride: int = 0, pos: int = 0, first: int = 0) -> list[int]:
    """An array whose rows follow the beams (BEAM_ACT, BEAM_STATE, BEAM_KV)."""
    return cmd(OP_BEAM_MOVE, kind | (n_part << 8), off, row_stride, part_stride, n, parent, n_beam | (n_group << 8)) + cmd(pos, first)


def beam_next(tok: int, pos: int, out: int, cap: int, n_seq: int) -> list[int]:
    return cmd(OP_BEAM_NEXT, tok, pos, out, cap, n_seq)


def fill(n: int, y: int, value: float) -> list[int]:
    return cmd(OP_FILL, n, y, fbits(value))


def gemm(fmt: int, rows: int, cols: int, w_off: int, x_off: int, y_off: int, n_tok: int, x_stride: int,
         y_stride: int, flags: int = 0, res_off: int = 0, res_stride: int = 0, norm_w: int = 0, eps: float = 0.0,
         norm_flags: int = 0) -> list[int]:
    """Batched GEMV over n_tok token rows (x_stride / y_stride floats apart); norm_flags NORM_DEFER folds a per-token
    RMS norm (weight at norm_w unless NORM_NO_WEIGHT) into the activation quantization."""
    out = cmd(OP_GEMM, fmt | flags, rows, cols, w_off & 0xFFFFFFFF, w_off >> 32, x_off, y_off)
    out += cmd(n_tok, x_stride, y_stride, res_off, res_stride, norm_w, fbits(eps), norm_flags)
    return out


# ---------------------------------------------------------------------------------------------------------------
_hip = None
_synth = None


class Kv4(C.Structure):  # gemvq_kv4
    """A 4-bit KV cache on device memory: its address (kv4_bytes() bytes) and sizes."""
    _fields_ = [("data", C.c_void_p)] + [(n, C.c_int32) for n in ("n_seq", "n_ctx", "n_head_kv", "head_dim")]


class BeamArray(C.Structure):  # gemvq_beam_array
    """An array whose rows follow the beams: its address, strides and units in bytes (gemvq_hip.h)."""
    _fields_ = [("data", C.c_void_p), ("row_stride", C.c_uint64), ("part_stride", C.c_uint64), ("n_part", C.c_uint32),
                ("first", C.c_uint32), ("count", C.c_uint32), ("unit_bytes", C.c_uint32), ("unit_len", C.c_uint32),
                ("used", C.c_void_p), ("used_stride", C.c_int32)]


class RopeRows(C.Structure):  # gemvq_rope_rows
    """Rows of heads that rope_static turns: addresses, strides in floats, heads a row."""
    _fields_ = [("x", C.c_void_p), ("y", C.c_void_p), ("x_row", C.c_int64), ("x_head", C.c_int64), ("y_row", C.c_int64),
                ("y_head", C.c_int64), ("n_head", C.c_int32)]


class LaunchStat(C.Structure):  # gemvq_launch_stat
    _fields_ = [("name", C.c_char * 40), ("first_cmd", C.c_int32), ("n_cmds", C.c_int32), ("bytes", C.c_uint64),
                ("us", C.c_double)]


def _c_fn(lib, name, res, *args):
    f = getattr(lib, name)
    f.restype = res
    f.argtypes = list(args)
    return f


def hip_lib() -> C.CDLL:
    """Loads libgemvq_hip.so (raises if it has not been built)."""
    global _hip
    if _hip is None:
        if not os.path.exists(HIP_LIB_PATH):
            raise RuntimeError(f"{HIP_LIB_PATH} is missing: build it first (python __graft_entry__.py or build.py)")
        lib = C.CDLL(HIP_LIB_PATH)
        vp, u64p = C.c_void_p, C.POINTER(C.c_uint64)
        _c_fn(lib, "gemvq_ctx_create", vp, C.c_int, C.c_size_t, C.c_size_t, C.c_size_t)
        _c_fn(lib, "gemvq_ctx_destroy", None, vp)
        _c_fn(lib, "gemvq_last_error", C.c_char_p, vp)
        _c_fn(lib, "gemvq_features", None, vp, C.POINTER(C.c_uint32))
        _c_fn(lib, "gemvq_upload_weight", C.c_int, vp, C.c_int, C.c_int, C.c_int, vp, u64p)
        _c_fn(lib, "gemvq_weight_bytes_used", C.c_uint64, vp)
        _c_fn(lib, "gemvq_repack", C.c_int, C.c_int, C.c_int, C.c_int, vp, vp)
        _c_fn(lib, "gemvq_unpack", C.c_int, C.c_int, C.c_int, C.c_int, vp, vp)
        _c_fn(lib, "gemvq_act_write", C.c_int, vp, C.c_size_t, vp, C.c_size_t)
        _c_fn(lib, "gemvq_act_read", C.c_int, vp, C.c_size_t, vp, C.c_size_t)
        _c_fn(lib, "gemvq_state_write", C.c_int, vp, C.c_size_t, vp, C.c_size_t)
        _c_fn(lib, "gemvq_state_read", C.c_int, vp, C.c_size_t, vp, C.c_size_t)
        _c_fn(lib, "gemvq_state_clear", C.c_int, vp)
        _c_fn(lib, "gemvq_set_kv_type", C.c_int, vp, C.c_int)
        _c_fn(lib, "gemvq_kv_create", C.c_int, vp, C.c_int, C.c_int, C.c_int)
        _c_fn(lib, "gemvq_kv_read", C.c_int, vp, C.c_int, C.c_int, C.c_int, vp, vp)
        _c_fn(lib, "gemvq_kv_clear", C.c_int, vp)
        _c_fn(lib, "gemvq_run", C.c_int, vp, C.POINTER(C.c_uint32), C.c_uint)
        _c_fn(lib, "gemvq_graph_create", C.c_int, vp, C.POINTER(C.c_uint32), C.c_uint, C.POINTER(C.c_int))
        _c_fn(lib, "gemvq_graph_replay", C.c_int, vp, C.c_int, C.c_int)
        _c_fn(lib, "gemvq_graph_destroy", C.c_int, vp, C.c_int)
        _c_fn(lib, "gemvq_sync", C.c_int, vp)
        _c_fn(lib, "gemvq_set_wait_timeout", C.c_int, vp, C.c_uint)
        _c_fn(lib, "gemvq_usable", C.c_int, vp)
        _c_fn(lib, "gemvq_last_launch_count", C.c_int, vp)
        _c_fn(lib, "gemvq_debug_blocksums", C.c_int, vp, vp, C.c_size_t)
        _c_fn(lib, "gemvq_graph_time", C.c_int, vp, C.c_int, C.c_int, C.POINTER(C.c_double))
        _c_fn(lib, "gemvq_set_arith", C.c_int, vp, C.c_int)
        _c_fn(lib, "gemvq_profile", C.c_int, vp, C.POINTER(C.c_uint32), C.c_uint, C.c_int, C.c_void_p, C.c_int)
        _c_fn(lib, "gemvq_arith", C.c_int, vp)
        _c_fn(lib, "gemvq_cr_expf", C.c_float, C.c_float)
        _c_fn(lib, "gemvq_cr_logf", C.c_float, C.c_float)
        _c_fn(lib, "gemvq_crmath_hash", C.c_int, vp, C.c_int, u64p)
        i, i64, u64, kvp = C.c_int, C.c_int64, C.c_uint64, C.POINTER(Kv4)
        _c_fn(lib, "gemvq_kv4_bytes", u64, i, i, i, i)
        for name in ("gemvq_kv4_store_static", "gemvq_kv4_load_static"):
            _c_fn(lib, name, i, kvp, vp, vp, i64, i, vp, vp, vp)
        _c_fn(lib, "gemvq_kv4_attn_work", u64, kvp, i, i)
        _c_fn(lib, "gemvq_kv4_attn_static", i, kvp, vp, i64, i64, vp, i64, i, i, vp, vp, i, C.c_float, vp, u64, vp)
        _c_fn(lib, "gemvq_beam_work", u64, i, i, i)
        _c_fn(lib, "gemvq_beam_select_static", i, vp, i64, i, i, i, vp, vp, i, vp, vp, vp, vp, u64, vp)
        _c_fn(lib, "gemvq_beam_reorder_static", i, C.POINTER(BeamArray), i, vp, i, i, vp)
        f64 = C.c_double
        _c_fn(lib, "gemvq_kv4_attn_sink_work", u64, kvp, i, i)
        _c_fn(lib, "gemvq_kv4_attn_sink_static", i, kvp, vp, i64, i64, vp, i64, i, i, vp, vp, i, i, C.c_float, vp, u64, vp)
        _c_fn(lib, "gemvq_kv4_attn_shared_work", u64, kvp, kvp, i, i)
        _c_fn(lib, "gemvq_kv4_attn_shared_static", i, kvp, kvp, vp, vp, i64, i64, vp, i64, i, i, vp, vp, i, i, C.c_float, vp, u64, vp)
        _c_fn(lib, "gemvq_rope_freqs", i, i, f64, f64, i, f64, f64, vp, vp)
        _c_fn(lib, "gemvq_rope_static", i, C.POINTER(RopeRows), i, i, i, i, i, i, vp, vp, vp, vp)
        _c_fn(lib, "gemvq_draft_work", u64, i, i, i)
        _c_fn(lib, "gemvq_draft_verify_static", i, vp, i64, vp, i64, i, i, i, vp, vp, vp, f64, f64, vp, vp, vp, vp, u64, vp)
        _hip = lib
    return _hip


def synth_lib() -> C.CDLL:
    global _synth
    if _synth is None:
        if not os.path.exists(SYNTH_LIB_PATH):
            raise RuntimeError(f"{SYNTH_LIB_PATH} is missing: build it first")
        lib = C.CDLL(SYNTH_LIB_PATH)
        vp = C.c_void_p
        _c_fn(lib, "gqs_u64", C.c_uint64, C.c_uint64, C.c_uint64, C.c_uint64)
        _c_fn(lib, "gqs_normal", None, C.c_uint64, C.c_uint64, C.c_uint64, C.c_size_t, C.c_float, C.c_float, vp)
        _c_fn(lib, "gqs_uniform", None, C.c_uint64, C.c_uint64, C.c_uint64, C.c_size_t, C.c_float, C.c_float, vp)
        _c_fn(lib, "gqs_quantize", C.c_size_t, C.c_int, vp, C.c_int64, C.c_int64, vp)
        _c_fn(lib, "gqs_row_bytes", C.c_size_t, C.c_int, C.c_int64)
        _c_fn(lib, "gqs_matrix", C.c_size_t, C.c_int, C.c_int64, C.c_int64, C.c_uint64, C.c_uint64, C.c_float,
              C.c_float, vp, C.c_int)
        _synth = lib
    return _synth


def _ptr(a: np.ndarray) -> int:
    assert a.flags["C_CONTIGUOUS"]
    return a.ctypes.data


# ---------------------------------------------------------------------------------------------------------------
# synthetic data
def normal(seed: int, stream: int, n: int, mean: float = 0.0, std: float = 1.0, first: int = 0) -> np.ndarray:
    out = np.empty(n, dtype=np.float32)
    synth_lib().gqs_normal(seed, stream, first, n, mean, std, _ptr(out))
    return out


def uniform(seed: int, stream: int, n: int, lo: float, hi: float, first: int = 0) -> np.ndarray:
    out = np.empty(n, dtype=np.float32)
    synth_lib().gqs_uniform(seed, stream, first, n, lo, hi, _ptr(out))
    return out


def quantize(t: int, x: np.ndarray, rows: int, cols: int) -> np.ndarray:
    x = np.ascontiguousarray(x, dtype=np.float32)
    assert x.size == rows * cols
    out = np.empty(rows * row_bytes(t, cols), dtype=np.uint8)
    if synth_lib().gqs_quantize(t, _ptr(x), rows, cols, _ptr(out)) != out.size:
        raise ValueError("quantize: unsupported type or shape")
    return out


def matrix(t: int, rows: int, cols: int, seed: int, stream: int, std: float = 0.02, mean: float = 0.0,
           threads: int = 0) -> np.ndarray:
    """rows x cols from N(mean, std^2) quantized to type t (GGUF bytes), generated in parallel."""
    threads = threads or min(16, os.cpu_count() or 1)
    out = np.empty(rows * row_bytes(t, cols), dtype=np.uint8)
    if synth_lib().gqs_matrix(t, rows, cols, seed, stream, mean, std, _ptr(out), threads) != out.size:
        raise ValueError("matrix: unsupported type or shape")
    return out


def repack(t: int, rows: int, cols: int, gguf: np.ndarray) -> np.ndarray:
    out = np.empty_like(gguf)
    if hip_lib().gemvq_repack(t, rows, cols, _ptr(gguf), _ptr(out)) != 0:
        raise ValueError("repack: bad type or shape")
    return out


def unpack(t: int, rows: int, cols: int, packed: np.ndarray) -> np.ndarray:
    out = np.empty_like(packed)
    if hip_lib().gemvq_unpack(t, rows, cols, _ptr(packed), _ptr(out)) != 0:
        raise ValueError("unpack: bad type or shape")
    return out


# ---------------------------------------------------------------------------------------------------------------
class GemvqError(RuntimeError):
    pass


# ---------------------------------------------------------------------------------------------------------------
# Operators on caller-owned device memory (gemvq_hip.h): pointers are addresses (a tensor's data_ptr(), say) on the
# current device, stream is a hipStream_t's value (0: the null stream). A program that uses torch imports it before the
# library is loaded, so that both work on one HIP runtime.
def _ok(st: int, what: str) -> None:
    if st:
        raise GemvqError(f"{what}: " + ("bad argument" if st == EINVAL else f"status {st}"))


def kv4_bytes(n_seq: int, n_ctx: int, n_head_kv: int, head_dim: int) -> int:
    """Bytes of a 4-bit KV cache (0: sizes that are not served)."""
    return hip_lib().gemvq_kv4_bytes(n_seq, n_ctx, n_head_kv, head_dim)


def kv4_store_static(kv: Kv4, k: int, v: int, row_stride: int, n_tok: int, pos: int, num: int = 0, stream: int = 0) -> None:
    """Stores the tokens' keys and values at positions pos[s] + t."""
    _ok(hip_lib().gemvq_kv4_store_static(kv, k, v, row_stride, n_tok, pos, num, stream), "kv4 store")


def kv4_load_static(kv: Kv4, k: int, v: int, row_stride: int, n_tok: int, pos: int, num: int = 0, stream: int = 0) -> None:
    """Reads the keys and values at positions pos[s] + t as FP32."""
    _ok(hip_lib().gemvq_kv4_load_static(kv, k, v, row_stride, n_tok, pos, num, stream), "kv4 load")


def kv4_attn_work(kv: Kv4, n_tok: int, n_head: int) -> int:
    """Bytes of workspace of kv4_attn_static."""
    return hip_lib().gemvq_kv4_attn_work(kv, n_tok, n_head)


def kv4_attn_static(kv: Kv4, q: int, q_stride: int, q_head_stride: int, y: int, y_stride: int, n_tok: int, n_head: int,
                    pos: int, num: int = 0, window: int = 0, scale: float = 1.0, work: int = 0, work_bytes: int = 0,
                    stream: int = 0) -> None:
    """Attention of the tokens at positions pos[s] + t over the cache (their own keys and values stored before)."""
    _ok(hip_lib().gemvq_kv4_attn_static(kv, q, q_stride, q_head_stride, y, y_stride, n_tok, n_head, pos, num, window, scale,
                                        work, work_bytes, stream), "kv4 attention")


def kv4_attn_sink_work(kv: Kv4, n_tok: int, n_head: int) -> int:
    """Bytes of workspace of kv4_attn_sink_static, and of its calls of smaller sizes (0: sizes that are not served)."""
    return hip_lib().gemvq_kv4_attn_sink_work(kv, n_tok, n_head)


def kv4_attn_sink_static(kv: Kv4, q: int, q_stride: int, q_head_stride: int, y: int, y_stride: int, n_tok: int, n_head: int,
                         pos: int, num: int = 0, window: int = 0, sinks: int = 0, scale: float = 1.0, work: int = 0,
                         work_bytes: int = 0, stream: int = 0) -> None:
    """Attention over the last `window` positions and the first `sinks`."""
    _ok(hip_lib().gemvq_kv4_attn_sink_static(kv, q, q_stride, q_head_stride, y, y_stride, n_tok, n_head, pos, num, window, sinks,
                                             scale, work, work_bytes, stream), "kv4 attention with sinks")


def kv4_attn_shared_work(kv: Kv4, prefix: Kv4, n_tok: int, n_head: int) -> int:
    """Bytes of workspace of kv4_attn_shared_static, and of its calls of smaller sizes (0: sizes that are not served)."""
    return hip_lib().gemvq_kv4_attn_shared_work(kv, prefix, n_tok, n_head)


def kv4_attn_shared_static(kv: Kv4, prefix: Kv4, prefix_len: int, q: int, q_stride: int, q_head_stride: int, y: int, y_stride: int,
                           n_tok: int, n_head: int, pos: int, num: int = 0, window: int = 0, sinks: int = 0, scale: float = 1.0,
                           work: int = 0, work_bytes: int = 0, stream: int = 0) -> None:
    """Attention of groups of sequences, each over its group's prefix and its own cache behind it."""
    _ok(hip_lib().gemvq_kv4_attn_shared_static(kv, prefix, prefix_len, q, q_stride, q_head_stride, y, y_stride, n_tok, n_head, pos,
                                               num, window, sinks, scale, work, work_bytes, stream), "kv4 attention with a prefix")


def beam_work(n_group: int, n_beam: int, n_vocab: int) -> int:
    """Bytes of workspace of beam_select_static (0: sizes that are not served)."""
    return hip_lib().gemvq_beam_work(n_group, n_beam, n_vocab)


def beam_select_static(logits: int, row_stride: int, n_vocab: int, n_group: int, n_beam: int, score: int, last: int, eos: int,
                       score_out: int, token: int, parent: int, work: int, work_bytes: int, stream: int = 0) -> None:
    """The n_beam best continuations of each group's beams: score, token and parent beam, in descending order."""
    _ok(hip_lib().gemvq_beam_select_static(logits, row_stride, n_vocab, n_group, n_beam, score, last, eos, score_out, token,
                                           parent, work, work_bytes, stream), "beam selection")


def beam_reorder_static(arrays, parent: int, n_group: int, n_beam: int, stream: int = 0) -> None:
    """In each of the arrays (BeamArray), row i of every group becomes a copy of its row parent[i]."""
    if not isinstance(arrays, C.Array):
        arrays = (BeamArray * len(arrays))(*arrays)
    _ok(hip_lib().gemvq_beam_reorder_static(arrays, len(arrays), parent, n_group, n_beam, stream), "beam reordering")


def rope_freqs(n_rot: int, base: float, factor: float = 1.0, yarn_ctx: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
               factors=None) -> np.ndarray:
    """The table of rope_static (turns per position of each pair, then the magnitude), to be copied to the device."""
    if factors is not None:
        factors = np.ascontiguousarray(factors, dtype=np.float64)
        if factors.size != n_rot // 2:
            raise GemvqError("rope table: a factor for each pair")
    out = np.empty(max(n_rot // 2, 0) + 1, dtype=np.float64)
    _ok(hip_lib().gemvq_rope_freqs(n_rot, base, factor, yarn_ctx, beta_fast, beta_slow, None if factors is None else _ptr(factors),
                                   _ptr(out)), "rope table")
    return out


def rope_static(arrays, n_seq: int, n_tok: int, head_dim: int, n_rot: int, layout: int, freqs: int, pos: int, num: int = 0,
                stream: int = 0) -> None:
    """Rotary positions pos[s] + t of the arrays' (RopeRows) heads."""
    if not isinstance(arrays, C.Array):
        arrays = (RopeRows * len(arrays))(*arrays)
    _ok(hip_lib().gemvq_rope_static(arrays, len(arrays), n_seq, n_tok, head_dim, n_rot, layout, freqs, pos, num, stream), "rope")


def draft_work(n_seq: int, n_draft: int, n_vocab: int) -> int:
    """Bytes of workspace of draft_verify_static, and of its calls of smaller sizes (0: sizes that are not served)."""
    return hip_lib().gemvq_draft_work(n_seq, n_draft, n_vocab)


def draft_verify_static(target: int, target_stride: int, draft: int, draft_stride: int, n_vocab: int, n_seq: int, n_draft: int,
                        token: int, num: int, uniform: int, temperature: float, draft_temperature: float, n_accept: int, out: int,
                        logp: int, work: int, work_bytes: int, stream: int = 0) -> None:
    """How many of the drafted tokens stand, and the token behind them."""
    _ok(hip_lib().gemvq_draft_verify_static(target, target_stride, draft, draft_stride, n_vocab, n_seq, n_draft, token, num, uniform,
                                            temperature, draft_temperature, n_accept, out, logp, work, work_bytes, stream),
        "draft verification")


class Context:
    """One device context: activation buffer (floats), weight arena, GDN state rows, KV buffers, graphs."""

    def __init__(self, act_floats: int = 1 << 22, weight_bytes: int = 1 << 28, state_rows: int = 0, device: int = 0):
        self.lib = hip_lib()
        self.h = self.lib.gemvq_ctx_create(device, act_floats, weight_bytes, state_rows)
        if not self.h:
            raise GemvqError(self.lib.gemvq_last_error(None).decode())
        self.act_floats = act_floats

    def close(self) -> None:
        if self.h:
            self.lib.gemvq_ctx_destroy(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def error(self) -> str:
        return self.lib.gemvq_last_error(self.h).decode()

    def _check(self, st: int, what: str) -> int:
        if st < 0:
            raise GemvqError(f"{what}: status {st}: {self.error()}")
        return st

    def features(self) -> tuple[int, int]:
        out = (C.c_uint32 * 2)()
        self.lib.gemvq_features(self.h, out)
        return int(out[0]), int(out[1])

    def upload(self, t: int, rows: int, cols: int, gguf: np.ndarray) -> int:
        gguf = np.ascontiguousarray(gguf, dtype=np.uint8)
        assert gguf.size == rows * row_bytes(t, cols)
        off = C.c_uint64()
        self._check(self.lib.gemvq_upload_weight(self.h, t, rows, cols, _ptr(gguf), C.byref(off)), "upload")
        return int(off.value)

    def write(self, off: int, data: np.ndarray) -> None:
        data = np.ascontiguousarray(data)
        assert data.dtype.itemsize == 4
        self._check(self.lib.gemvq_act_write(self.h, off, _ptr(data), data.size), "act write")

    def read(self, off: int, n: int, dtype=np.float32) -> np.ndarray:
        out = np.empty(n, dtype=dtype)
        self._check(self.lib.gemvq_act_read(self.h, off, _ptr(out), n), "act read")
        return out

    def state_write(self, row: int, data: np.ndarray) -> None:
        data = np.ascontiguousarray(data, dtype=np.float32)
        assert data.size % 128 == 0
        self._check(self.lib.gemvq_state_write(self.h, row, _ptr(data), data.size // 128), "state write")

    def state_read(self, row: int, rows: int) -> np.ndarray:
        out = np.empty(rows * 128, dtype=np.float32)
        self._check(self.lib.gemvq_state_read(self.h, row, _ptr(out), rows), "state read")
        return out

    def set_kv_type(self, kind: int) -> None:
        """KV_F16 (default) or KV_Q4_0: what the KV buffers created from now on hold."""
        self._check(self.lib.gemvq_set_kv_type(self.h, kind), "set kv type")

    def kv_create(self, n_ctx: int, n_head_kv: int, head_dim: int) -> int:
        return self._check(self.lib.gemvq_kv_create(self.h, n_ctx, n_head_kv, head_dim), "kv create")

    def kv_read(self, kv: int, pos0: int, npos: int, row: int) -> tuple[np.ndarray, np.ndarray]:
        k = np.empty(npos * row, dtype=np.uint16)
        v = np.empty(npos * row, dtype=np.uint16)
        self._check(self.lib.gemvq_kv_read(self.h, kv, pos0, npos, _ptr(k), _ptr(v)), "kv read")
        return k, v

    @staticmethod
    def _words(cmds) -> tuple[np.ndarray, int]:
        w = np.ascontiguousarray(np.asarray(cmds, dtype=np.uint64).astype(np.uint32).ravel())
        assert w.size % 8 == 0
        return w, w.size // 8

    def run(self, cmds) -> int:
        """Runs a command list; returns 0 or the 1-based index of the first invalid command; raises on errors."""
        w, n = self._words(cmds)
        return self._check(self.lib.gemvq_run(self.h, w.ctypes.data_as(C.POINTER(C.c_uint32)), n), "run")

    def graph(self, cmds) -> int:
        w, n = self._words(cmds)
        g = C.c_int(-1)
        st = self.lib.gemvq_graph_create(self.h, w.ctypes.data_as(C.POINTER(C.c_uint32)), n, C.byref(g))
        if st != 0:
            raise GemvqError(f"graph create: status {st}: {self.error()}")
        return g.value

    def replay(self, g: int, times: int = 1) -> None:
        self._check(self.lib.gemvq_graph_replay(self.h, g, times), "replay")

    def graph_time_us(self, g: int, times: int) -> float:
        us = C.c_double()
        self._check(self.lib.gemvq_graph_time(self.h, g, times, C.byref(us)), "graph time")
        return us.value

    def sync(self) -> None:
        self._check(self.lib.gemvq_sync(self.h), "sync")

    def set_wait_timeout(self, ms: int) -> None:
        """Bound of every wait for the device (a timed-out wait makes the context unusable)."""
        self._check(self.lib.gemvq_set_wait_timeout(self.h, ms), "wait timeout")

    def usable(self) -> bool:
        return bool(self.lib.gemvq_usable(self.h))

    def launch_count(self) -> int:
        return self.lib.gemvq_last_launch_count(self.h)

    def set_arith(self, arith: int) -> None:
        """Arithmetic of the lists compiled from now on: ARITH_CANONICAL (default) or ARITH_REFERENCE (the reference's
        CPU arithmetic, gemvq_hip.h)."""
        self._check(self.lib.gemvq_set_arith(self.h, arith), "set arith")

    def arith(self) -> int:
        return self.lib.gemvq_arith(self.h)

    def profile(self, cmds, reps: int = 1) -> list[dict]:
        """The launches the list compiles to, each timed on the stream with HIP events (gemvq_profile: the median
        over reps repetitions of the list): name, first command, HBM bytes (algorithmic), microseconds."""
        w, n = self._words(cmds)
        out = (LaunchStat * 4096)()
        got = self.lib.gemvq_profile(self.h, w.ctypes.data_as(C.POINTER(C.c_uint32)), n, reps, out, 4096)
        if got < 0:
            raise GemvqError(f"profile: {got}: {self.error()}")
        return [dict(name=out[i].name.decode(), first=out[i].first_cmd, bytes=int(out[i].bytes), us=out[i].us)
                for i in range(got)]

    def crmath_hash(self, fn: int) -> np.ndarray:
        """The device's correctly rounded exp (fn 0) or log (fn 1) over every binary32 input, as 4096 block hashes."""
        out = np.zeros(4096, dtype=np.uint64)
        self._check(self.lib.gemvq_crmath_hash(self.h, fn, out.ctypes.data_as(C.POINTER(C.c_uint64))), "crmath hash")
        return out

    def debug_blocksums(self, out: np.ndarray) -> None:
        assert out.dtype == np.int32 and out.flags["C_CONTIGUOUS"]
        self._check(self.lib.gemvq_debug_blocksums(self.h, _ptr(out), out.size), "debug blocksums")
