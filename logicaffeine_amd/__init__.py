"""logicaffeine_amd -- Python view of liblgx, the MI355X back-end of the Q8
LLM-decode hot path.

Every compute call goes through the C ABI in ``include/lgx.h`` (liblgx.so ->
hipModuleLaunchKernel on lgx_kernels.hsaco).  There is no CPU or PyTorch
fallback: if the library or its code object is missing, :class:`Context`
raises.  torch is used only for device memory and the current stream.

The loader mirrors the reference's AOT tier (load a built module, resolve its
``extern "C"`` symbols, keep it alive, count calls;
crates/logicaffeine_compile/src/vm/aot_tier.rs:86-111), and errors surface as
:class:`LgxError` carrying the ``lgx_status`` and ``lgx_last_error()`` text
(crates/logicaffeine_compile/src/codegen/ffi.rs:196-258).
"""
from __future__ import annotations

import ctypes as C
import os
import weakref

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "liblgx.so")
HSACO_PATH = os.path.join(HERE, "lgx_kernels.hsaco")

Q8_ROWMAJOR = 0
Q8_T16 = 1
Q8_RANGE_BLOCKS = 32

STATUS_NAMES = {
    0: "LGX_OK", 1: "LGX_ERROR", 2: "LGX_INVALID_ARGUMENT", 3: "LGX_NULL_POINTER",
    4: "LGX_OUT_OF_BOUNDS", 5: "LGX_MODULE_LOAD_FAILED", 6: "LGX_INVALID_HANDLE",
    8: "LGX_INTERNAL_PANIC", 9: "LGX_OUT_OF_MEMORY", 10: "LGX_HIP_ERROR",
    11: "LGX_NO_DEVICE", 12: "LGX_UNSUPPORTED",
}

# Exported symbols and their C signatures (include/lgx.h).
_P = C.c_void_p
_I32 = C.c_int32
SIGNATURES = {
    "lgx_abi_version": (C.c_uint32, []),
    "lgx_version": (C.c_char_p, []),
    "lgx_last_error": (C.c_char_p, []),
    "lgx_clear_error": (None, []),
    "lgx_ctx_create": (C.c_int, [_I32, C.c_char_p, C.POINTER(_P)]),
    "lgx_ctx_destroy": (C.c_int, [_P]),
    "lgx_ctx_launch_count": (C.c_uint64, [_P]),
    "lgx_ctx_arch": (C.c_char_p, [_P]),
    "lgx_ctx_set_kernel_timing": (C.c_int, [_P, _I32]),
    "lgx_ctx_kernel_stats": (C.c_int, [_P, C.c_char_p, C.POINTER(C.c_uint64),
                                       C.POINTER(C.c_double)]),
    "lgx_q8_scale_count": (C.c_size_t, [_I32, _I32]),
    "lgx_q8_repack_t16": (C.c_int, [_P, _P, _P, _I32, _I32, _P, _P, _P]),
    "lgx_q8_unpack_t16": (C.c_int, [_P, _P, _P, _I32, _I32, _P, _P, _P]),
    "lgx_quantize_q8_0": (C.c_int, [_P, _P, _I32, _I32, _P, _P, _P]),
    "lgx_q8_gemv_f32": (C.c_int, [_P, _P, _P, _P, _P]),
    "lgx_q8q8_gemv": (C.c_int, [_P, _P, _P, _P, _P, _P, _P]),
    "lgx_q8_gemm": (C.c_int, [_P, _P, _P, _P, _I32, _P, _P]),
    "lgx_q8_gemm_noalloc": (C.c_int, [_P, _P, _P, _P, _I32, _P, _P]),
    "lgx_q8q8_gemv_quantize": (C.c_int, [_P, _P, _P, _P, _P, _P, _P]),
    "lgx_q8q8_gemv_quantize_group": (C.c_int, [_P, _I32, _P, _P, _P, _P]),
    "lgx_q8_gemm_quantize_group": (C.c_int, [_P, _I32, _P, _P, _I32, _P, _P]),
    "lgx_q8_range_count": (_I32, [_I32]),
    "lgx_q8q8_gemv_quantize_partials": (C.c_int, [_P, _P, _P, _P, _P, _P, _P]),
    "lgx_q8_gemm_partials": (C.c_int, [_P, _P, _P, _P, _I32, _P, _P]),
    "lgx_q8_range_combine": (C.c_int, [_P, _P, _I32, C.c_int64, _P, _P]),
    "lgx_gqa_decode_attn": (C.c_int, [_P, _P, _P, _P, _P, _P, _I32, _I32, _I32, _I32, _I32,
                                      _I32, _I32, _P, _P]),
    "lgx_gqa_prefill_attn": (C.c_int, [_P, _P, _P, _P, _P, _P, _I32, _I32, _I32, _I32, _I32,
                                       _I32, _I32, _I32, _P, _P]),
    "lgx_gqa_prefill_attn_fast": (C.c_int, [_P, _P, _P, _P, _P, _P, _I32, _I32, _I32, _I32,
                                            _I32, _I32, _I32, _I32, _P, _P]),
    "lgx_embed_f16": (C.c_int, [_P, _P, _P, _I32, _I32, _I32, _P, _P]),
    "lgx_rmsnorm_quant": (C.c_int, [_P, _P, _P, _I32, _I32, C.c_float, _P, _P, _P, _P]),
    "lgx_add_rmsnorm_quant": (C.c_int, [_P, _P, _I32, _P, _P, _I32, _I32, C.c_float, _P, _P, _P,
                                        _P]),
    "lgx_rope_kv_append": (C.c_int, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I32, _I32, _I32,
                                     _I32, _I32, _I32, _I32, _P]),
    "lgx_swiglu_quant": (C.c_int, [_P, _P, _I32, _I32, _P, _P, _P, _P]),
    "lgx_lm_head_f16": (C.c_int, [_P, _P, _P, _I32, _I32, _I32, _P, _P]),
    "lgx_f16_t64_count": (C.c_int64, [_I32, _I32]),
    "lgx_f16_repack_t64": (C.c_int, [_P, _P, _I32, _I32, _P, _P]),
    "lgx_lm_head_f16_t64": (C.c_int, [_P, _P, _P, _I32, _I32, _I32, _P, _P]),
    "lgx_lm_head_rowconst": (C.c_int, [_P, _P, _I32, _I32, _P, _P]),
    "lgx_lm_head_argmax_f16": (C.c_int, [_P, _P, _P, _P, _P, _I32, _I32, _I32, _P, _P, _P]),
    "lgx_argmax": (C.c_int, [_P, _P, _I32, _I32, _P, _P]),
    "lgx_sample": (C.c_int, [_P, _P, _I32, _I32, _I32, C.c_float, C.c_float, C.c_uint64, _P, _P,
                             _P]),
    "lgx_model_set_sampling": (C.c_int, [_P, C.c_float, _I32, C.c_float, C.c_uint64]),
    "lgx_model_set_prefill_mode": (C.c_int, [_P, _I32]),
    "lgx_model_create": (C.c_int, [_P, _P, C.c_uint64, C.POINTER(_P)]),
    "lgx_gguf_config": (C.c_int, [C.c_char_p, _I32, _I32, _P]),
    "lgx_model_load_gguf": (C.c_int, [_P, C.c_char_p, _I32, _I32, C.POINTER(_P)]),
    "lgx_model_config": (C.c_int, [_P, _P]),
    "lgx_model_destroy": (C.c_int, [_P]),
    "lgx_model_reset": (C.c_int, [_P, _P]),
    "lgx_qwen_decode_step": (C.c_int, [_P, _I32, _P, _P]),
    "lgx_qwen_prefill": (C.c_int, [_P, _I32, _I32, _P, _P, _P]),
    "lgx_qwen_generate": (C.c_int, [_P, _I32, _P, _I32, _P, _P]),
    "lgx_model_tensor": (C.c_int, [_P, _I32, _I32, C.POINTER(_P), C.POINTER(C.c_size_t)]),
    "lgx_qwen_logits": (C.c_int, [_P, _I32, _P, _P]),
    "lgx_rope_tables": (C.c_int, [_I32, _I32, C.c_double, _P, _P, _P]),
    "lgx_rope_kv_append_i8": (C.c_int, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _I32, _I32, _I32, _I32, _P]),
    "lgx_kv_read_i8": (C.c_int, [_P, _P, _P, _P, _I32, _I32, _I32, _P, _P, _P]),
    "lgx_gqa_decode_attn_i8": (C.c_int, [_P, _P, _P, _P, _P, _I32, _I32, _I32, _I32, _P, _P, _P]),
    "lgx_gqa_prefill_attn_i8": (C.c_int, [_P, _P, _P, _P, _P, _P, _I32, _I32, _I32, _I32, _I32, _P, _P, _P]),
    "lgx_tree_plan": (C.c_int, [_P, _P, _P, _I32, _I32, _P, _P, _P]),
    "lgx_rope_kv_append_rows": (C.c_int, [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I32, _I32, _I32, _I32, _P]),
    "lgx_gqa_tree_attn": (C.c_int, [_P, _P, _P, _P, _P, _P, _P, _P, _I32, _I32, _I32, _I32, _I32, _P, _P, _P]),
    "lgx_tree_accept": (C.c_int, [_P, _P, _P, _P, _P, _P, _I32, _I32, _P, _P, _P, _P, _P]),
    "lgx_kv_keep": (C.c_int, [_P, _P, _I32, _P, _P, _P, _P, _I32, _I32, _I32, _P]),
    "lgx_sample_filtered": (C.c_int, [_P, _P, C.c_int64, _I32, _I32, _P, _P, _P, _P, _P, _P, _P, _P]),
    "lgx_pages_fork": (C.c_int, [_P, _P, _P, _P, _P, _P, _I32, _I32, _I32, _P]),
    "lgx_pages_reserve": (C.c_int, [_P, _P, _P, _P, _P, _I32, _I32, _P, _P, _P, _P]),
    "lgx_pages_copy": (C.c_int, [_P, _P, _I32, _I32, _P, _P, _I32, _P]),
    "lgx_pages_free": (C.c_int, [_P, _P, _P, _P, _I32, _I32, _P]),
}

# Model shapes of the decode benchmarks (random-init Qwen2.5-0.5B / -7B shaped
# Q8_0 models): keys as lgx.Model's cfg.
QWEN_SHAPES = {
    "0.5b": dict(n_layers=24, hidden=896, inter=4864, n_heads=14, n_kv=2, head_dim=64,
                 vocab=151936, tied=1),
    "7b": dict(n_layers=28, hidden=3584, inter=18944, n_heads=28, n_kv=4, head_dim=128,
               vocab=152064, tied=0),
}


def qwen_shape(name: str, max_batch: int, max_seq: int, emb_sigma: float = 0.002) -> dict:
    """cfg dict for lgx.Model: shape `name` with RMSNorm eps 1e-6, RoPE theta 1e6."""
    return dict(QWEN_SHAPES[name], max_batch=max_batch, max_seq=max_seq, eps=1e-6, theta=1e6,
                emb_sigma=emb_sigma)


def decode_step_bytes(cfg: dict, B: int, context: float) -> float:
    """Algorithmic HBM bytes of one greedy decode step of B sequences whose
    attention spans `context` cached tokens on average (the new token
    included): Q8_0 weights (1.0625 B/weight), the lm_head (binary16 tied
    embedding or Q8_0), the K/V cache read and the new K/V rows written."""
    H, I, d = cfg["hidden"], cfg["inter"], cfg["head_dim"]
    hq, hkv, L, V = cfg["n_heads"], cfg["n_kv"], cfg["n_layers"], cfg["vocab"]
    per_layer = ((hq + 2 * hkv) * d * H + H * hq * d + 2 * I * H + H * I) * 1.0625
    lm = V * H * (2.0 if cfg["tied"] else 1.0625)
    kv_row = L * hkv * d * 2 * 2                    # K and V, binary16, all layers
    return L * per_layer + lm + B * context * kv_row + B * kv_row


# Non-packed binary32 VALU lane operations per second of MI355X: 256 CUs x 4
# SIMDs x 16 lanes x 2.4 GHz (the published 157.3 TFLOP/s counts an FMA as
# two flops and packed FP32, which this build does not use).
VALU_LANE_OPS_PEAK = 256 * 4 * 16 * 2.4e9


def prefill_int8_ops(cfg: dict, B: int, P: int) -> float:
    """int8 MFMA operations (2 per multiply-add) of the Q8_0 products of the
    prefill of B prompts of P tokens: rows B x (P - 1) through the batched
    chunks (the last layer of a chunk runs its QKV product only), the last
    position of every prompt through the decode step, and the untied lm_head
    for those B rows (the tied lm_head is a binary16 VALU chain)."""
    H, I, d = cfg["hidden"], cfg["inter"], cfg["head_dim"]
    hq, hkv, L, V = cfg["n_heads"], cfg["n_kv"], cfg["n_layers"], cfg["vocab"]
    qkv = (hq + 2 * hkv) * d * H
    full = qkv + H * hq * d + 2 * I * H + H * I
    rows = B * (P - 1)
    macs = rows * ((L - 1) * full + qkv) + B * L * full
    if not cfg["tied"]:
        macs += B * V * H
    return 2.0 * macs


def prefill_fast_flops(cfg: dict, B: int, P: int) -> tuple:
    """MFMA work of the fast prefill of B prompts of P tokens: (binary16
    flops, int8 operations).  binary16: the GEMMs of the batched rows
    B x (P - 1) (2 per multiply-add; the last layer of a chunk runs its qkv
    GEMM only) and the causal attention of layers 0 .. L - 2 (2 d per query
    head and attended token for the scores, 2 d for PV; the row at position
    p attends p + 1 tokens).  int8: the last position of every prompt
    through the exact decode step (and the untied Q8_0 lm_head)."""
    H, I, d = cfg["hidden"], cfg["inter"], cfg["head_dim"]
    hq, hkv, L, V = cfg["n_heads"], cfg["n_kv"], cfg["n_layers"], cfg["vocab"]
    qkv = (hq + 2 * hkv) * d * H
    full = qkv + H * hq * d + 2 * I * H + H * I
    rows = B * (P - 1)
    gemm = 2.0 * rows * ((L - 1) * full + qkv)
    att_rows = B * (P - 1) * P / 2.0
    attn = 4.0 * d * hq * att_rows * (L - 1)
    int8 = 2.0 * B * (L * full + (0 if cfg["tied"] else V * H))
    return gemm + attn, int8


def prefill_valu_ops(cfg: dict, B: int, P: int) -> float:
    """Essential VALU lane operations of the canonical prefill of B prompts of
    P tokens (rows B x (P - 1) through the batched chunks, the last position
    through the decode step): 2 per (row, output, 32-block) of every Q8_0
    product (cvt of the int32 block dot, chain FMA; the scale products come
    from a rank-1 f16 MFMA) and 1 per attention FMA (score chain over d and PV
    chain over the attended tokens, per query head).  The last layer of a
    batched chunk stops after its KV append (QKV product only)."""
    H, I, d = cfg["hidden"], cfg["inter"], cfg["head_dim"]
    hq, hkv, L, V = cfg["n_heads"], cfg["n_kv"], cfg["n_layers"], cfg["vocab"]
    qkv = (hq + 2 * hkv) * d * H / 32
    full = qkv + (H * hq * d + 2 * I * H + H * I) / 32
    rows = B * (P - 1)
    gemm = 2.0 * (rows * ((L - 1) * full + qkv) + B * L * full)
    gemm += B * V * H * (1.0 if cfg["tied"] else 3.0 / 32)
    # attention: row at position p attends p + 1 tokens (2d FMAs per head each)
    att_rows = B * (P - 1) * P / 2.0            # sum over p < P - 1 of (p + 1)
    attn = 2.0 * d * hq * (att_rows * (L - 1) + B * P * L)
    return gemm + attn


# Tensor ids of lgx_model_tensor.
MODEL_TENSORS = {"emb": 0, "lm_q": 1, "lm_d": 2, "qkv_q": 3, "qkv_d": 4, "o_q": 5, "o_d": 6,
                 "gu_q": 7, "gu_d": 8, "dn_q": 9, "dn_d": 10, "bias": 11, "k_pages": 12,
                 "v_pages": 13, "page_table": 14, "seq_len": 15, "hidden": 16,
                 "attn_norm": 17, "ffn_norm": 18, "out_norm": 19, "emb_q": 20, "emb_d": 21}


class LgxError(RuntimeError):
    def __init__(self, status: int, message: str):
        self.status = status
        self.status_name = STATUS_NAMES.get(status, str(status))
        super().__init__(f"{self.status_name}: {message}")


class Q8MatrixC(C.Structure):
    _fields_ = [("qs", _P), ("d", _P), ("n", _I32), ("k", _I32), ("layout", _I32)]


class QwenConfigC(C.Structure):
    """lgx_qwen_config."""
    _fields_ = [("n_layers", _I32), ("hidden", _I32), ("intermediate", _I32),
                ("n_heads", _I32), ("n_kv_heads", _I32), ("head_dim", _I32), ("vocab", _I32),
                ("tied_embedding", _I32), ("max_batch", _I32), ("max_seq", _I32),
                ("rms_eps", C.c_float), ("rope_theta", C.c_double), ("emb_sigma", C.c_double)]


class KvI8C(C.Structure):
    """lgx_kv_i8."""
    _fields_ = [("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("num_pages", _I32),
                ("hkv", _I32), ("d", _I32)]


class RopeC(C.Structure):
    """lgx_rope."""
    _fields_ = [("cos_t", _P), ("sin_t", _P), ("rot", _I32), ("interleaved", _I32), ("max_pos", _I32)]


class RopeScalingC(C.Structure):
    """lgx_rope_scaling."""
    _fields_ = [("kind", _I32), ("original_len", _I32), ("factor", C.c_double), ("slow", C.c_double),
                ("fast", C.c_double)]


class AttnOptsC(C.Structure):
    """lgx_attn_opts."""
    _fields_ = [("scale", C.c_float), ("softcap", C.c_float), ("window", _I32), ("slopes", _P)]


class KvF16C(C.Structure):
    """lgx_kv_f16."""
    _fields_ = [("k", _P), ("v", _P), ("num_pages", _I32), ("hkv", _I32), ("d", _I32)]


class PagePoolC(C.Structure):
    """lgx_page_pool."""
    _fields_ = [("ref", _P), ("num_pages", _I32)]


class PagePlaneC(C.Structure):
    """lgx_page_plane."""
    _fields_ = [("data", _P), ("page_bytes", C.c_int64)]


_lib = None


def lib() -> C.CDLL:
    """Load liblgx.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is missing: build it with `python -m logicaffeine_amd.build`")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _check(status: int) -> None:
    if status != 0:
        msg = lib().lgx_last_error()
        raise LgxError(status, msg.decode(errors="replace") if msg else "(no message)")


def _stream(torch, device):
    """hipStream_t of torch's current stream on `device`, as an integer.  The
    raw query (0.07 us) where torch has it: building the Stream object of
    torch.cuda.current_stream takes 2 us of a 7.3 us call."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device.index) if raw else torch.cuda.current_stream(device).cuda_stream


class Q8Matrix:
    """A Q8_0 weight matrix resident on the device in the tile layouts.

    ``qs`` is an int8 device tensor (T16 order, n*k bytes); ``d`` an int16
    device tensor holding the binary16 scale bits in S16 order
    (lgx_q8_scale_count(n, k) elements)."""

    def __init__(self, qs, d, n: int, k: int):
        self.qs, self.d, self.n, self.k = qs, d, n, k
        self._c = Q8MatrixC(qs.data_ptr(), d.data_ptr(), n, k, Q8_T16)

    @property
    def cstruct(self):
        return C.byref(self._c)

    @property
    def nbytes(self) -> int:
        return self.qs.numel() + 2 * self.d.numel()


def _tensor(name, x, dtype, shape, dev):
    """x, refused unless it is a contiguous tensor of that type and shape (None: any
    extent) on dev."""
    if x.dtype is not dtype or x.device != dev or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor on {dev}, not {x.dtype} on {x.device}")
    if x.shape != shape and (len(x.shape) != len(shape) or any(w is not None and w != n for w, n in zip(shape, x.shape))):
        raise ValueError(f"{name} has shape {tuple(x.shape)}, expected {tuple(shape)}")
    return x


class _Held:
    """What a C struct points to.  Attributes are given by the constructor and stay:
    the struct would go on naming the memory of a tensor that was put aside."""

    def _hold(self, **attributes):
        self.__dict__.update(attributes)

    def __setattr__(self, name, value):
        raise AttributeError(f"{type(self).__name__}.{name} cannot be set: make a new {type(self).__name__}")

    def __delattr__(self, name):
        raise AttributeError(f"{type(self).__name__}.{name} cannot be deleted")


class KvCacheI8(_Held):
    """An 8-bit paged KV cache (lgx_kv_i8): int8 K pages [pages][hkv][16][d] and V
    pages [pages][hkv][d][16], float32 scales [pages][hkv] for each."""

    def __init__(self, k, v, k_scale, v_scale):
        import torch as t

        if k.dim() != 4:
            raise ValueError(f"k has shape {tuple(k.shape)}, expected [pages][hkv][16][d]")
        n, hkv, _, d = k.shape
        _tensor("k", k, t.int8, (n, hkv, 16, d), k.device)
        _tensor("v", v, t.int8, (n, hkv, d, 16), k.device)
        _tensor("k_scale", k_scale, t.float32, (n, hkv), k.device)
        _tensor("v_scale", v_scale, t.float32, (n, hkv), k.device)
        self._hold(k=k, v=v, k_scale=k_scale, v_scale=v_scale, num_pages=n, hkv=hkv, d=d, device=k.device,
                   cstruct=C.byref(KvI8C(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n, hkv, d)))

    @classmethod
    def empty(cls, ctx: "Context", num_pages: int, hkv: int, d: int) -> "KvCacheI8":
        """A cache of zeros on ctx's device."""
        t = ctx.torch
        return cls(t.zeros((num_pages, hkv, 16, d), dtype=t.int8, device=ctx.dev),
                   t.zeros((num_pages, hkv, d, 16), dtype=t.int8, device=ctx.dev),
                   t.zeros((num_pages, hkv), dtype=t.float32, device=ctx.dev),
                   t.zeros((num_pages, hkv), dtype=t.float32, device=ctx.dev))


class KvCacheF16(_Held):
    """A binary16 paged KV cache (lgx_kv_f16): K and V pages [pages][hkv][16][d], both
    float16, or both int16 with its bits."""

    def __init__(self, k, v):
        import torch as t

        if k.dim() != 4 or k.dtype not in (t.float16, t.int16):
            raise ValueError(f"k is {k.dtype} {tuple(k.shape)}, expected float16 or int16 [pages][hkv][16][d]")
        n, hkv, _, d = k.shape
        _tensor("k", k, k.dtype, (n, hkv, 16, d), k.device)
        _tensor("v", v, k.dtype, (n, hkv, 16, d), k.device)
        c = KvF16C(k.data_ptr(), v.data_ptr(), n, hkv, d)
        self._hold(k=k, v=v, num_pages=n, hkv=hkv, d=d, device=k.device, where=str(k.device), raw=bytes(c),
                   cstruct=C.byref(c))

    @classmethod
    def empty(cls, ctx: "Context", num_pages: int, hkv: int, d: int) -> "KvCacheF16":
        """A cache of zeros on ctx's device."""
        t = ctx.torch
        return cls(*(t.zeros((num_pages, hkv, 16, d), dtype=t.float16, device=ctx.dev) for _ in range(2)))


class Rope(_Held):
    """Rotation of query and key heads (lgx_rope): cos / sin are float32 device
    tensors [positions][rot / 2], the first rot dimensions of a head are turned in
    pairs (i, i + rot / 2), or (2i, 2i + 1) when interleaved."""

    def __init__(self, cos, sin, interleaved: bool = False):
        import torch as t

        n, half = cos.shape
        _tensor("cos", cos, t.float32, (n, half), cos.device)
        _tensor("sin", sin, t.float32, (n, half), cos.device)
        self._hold(cos=cos, sin=sin, device=cos.device,
                   cstruct=C.byref(RopeC(cos.data_ptr(), sin.data_ptr(), 2 * half, int(interleaved), n)))

    @classmethod
    def tables(cls, ctx: "Context", max_pos: int, rot: int, theta: float = 1e6, interleaved: bool = False,
               scaling: str = "plain", factor: float = 1.0, original_len: int = 0, slow: float = 1.0,
               fast: float = 32.0) -> "Rope":
        """Tables of lgx_rope_tables on ctx's device; scaling: "plain", "linear",
        "base" or "parts"."""
        t = ctx.torch
        kinds = ("plain", "linear", "base", "parts")
        if scaling not in kinds:
            raise ValueError(f"scaling {scaling!r} is none of {kinds}")
        sc = RopeScalingC(kinds.index(scaling), original_len, factor, slow, fast)
        shape = (max(max_pos, 0), max(rot, 0) // 2)
        cos, sin = t.empty(shape, dtype=t.float32), t.empty(shape, dtype=t.float32)
        _check(lib().lgx_rope_tables(max_pos, rot, theta, C.byref(sc), cos.data_ptr(), sin.data_ptr()))
        return cls(cos.to(ctx.dev), sin.to(ctx.dev), interleaved)


class AttnOpts(_Held):
    """Options of the 8-bit cache's attention (lgx_attn_opts): scale 0 is
    1 / sqrt(d); softcap 0 and window 0 are none; slopes: float32 [hq]."""

    def __init__(self, scale: float = 0.0, softcap: float = 0.0, window: int = 0, slopes=None):
        if slopes is not None:
            import torch as t

            _tensor("slopes", slopes, t.float32, (None,), slopes.device)
        self._hold(slopes=slopes, cstruct=C.byref(AttnOptsC(scale, softcap, window, _ptr_or_none(slopes))))


class PagePool(_Held):
    """The holders of a cache's pages (lgx_page_pool): int32 [pages], 0 for a free page."""

    def __init__(self, ref):
        import torch as t

        _tensor("ref", ref, t.int32, (None,), ref.device)
        self._hold(ref=ref, num_pages=ref.shape[0], device=ref.device, cstruct=C.byref(PagePoolC(ref.data_ptr(), ref.shape[0])))

    @classmethod
    def empty(cls, ctx: "Context", num_pages: int) -> "PagePool":
        """A pool of free pages on ctx's device."""
        return cls(ctx.torch.zeros(num_pages, dtype=ctx.torch.int32, device=ctx.dev))


class PagePlanes(_Held):
    """The arrays that a page copy goes over: contiguous tensors [pages][...] of one
    device, such as every layer's K and V pages and an 8-bit cache's scales."""

    def __init__(self, tensors):
        tensors = tuple(tensors)
        if not tensors:
            raise ValueError("no planes")
        n, device = tensors[0].shape[0], tensors[0].device
        for x in tensors:
            _tensor("a plane", x, x.dtype, (n, *x.shape[1:]), device)
        array = (PagePlaneC * len(tensors))(*[PagePlaneC(x.data_ptr(), x[0].numel() * x.element_size()) for x in tensors])
        self._hold(tensors=tensors, num_pages=n, device=device, count=len(tensors), carray=array)


class Context:
    """One lgx_ctx: the loaded code object on one device."""

    def __init__(self, device: int = 0, hsaco: str | None = None):
        import torch

        self.torch = torch
        self.device = device
        self.dev = torch.device("cuda", device)
        self.where = str(self.dev)
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        h = C.c_void_p()
        _check(lib().lgx_ctx_create(device, hsaco.encode() if hsaco else None, C.byref(h)))
        self.handle = h
        self._models = weakref.WeakSet()   # live Models built on this ctx

    def close(self) -> None:
        """Destroy the ctx; Models still open on it are closed first
        (lgx_ctx_destroy refuses a ctx that live models still use)."""
        if self.handle:
            for m in list(self._models):
                m.close()
            _check(lib().lgx_ctx_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def launch_count(self) -> int:
        return int(lib().lgx_ctx_launch_count(self.handle))

    @property
    def arch(self) -> str:
        return lib().lgx_ctx_arch(self.handle).decode()

    def _s(self):
        raw = self._raw_stream
        return raw(self.device) if raw else _stream(self.torch, self.dev)

    def kernel_timing(self, enable: bool) -> None:
        """Time every launch by its own dispatch (fresh window when enabled)."""
        _check(lib().lgx_ctx_set_kernel_timing(self.handle, 1 if enable else 0))

    def kernel_stats(self, kernel_name: str):
        """(launch count, total ms) of `kernel_name` in the timing window."""
        n, ms = C.c_uint64(), C.c_double()
        _check(lib().lgx_ctx_kernel_stats(self.handle, kernel_name.encode(), C.byref(n),
                                          C.byref(ms)))
        return int(n.value), float(ms.value)

    # ---- layout ----------------------------------------------------------
    def repack_t16(self, qs_rowmajor, d_rowmajor):
        """Row-major quants [n][k] + scales [n][k/32] -> (T16 quants, S16 scales)."""
        t = self.torch
        n, k = qs_rowmajor.shape
        out = t.empty(n * k, dtype=t.int8, device=self.dev)
        dout = t.empty(max(1, lib().lgx_q8_scale_count(n, k)), dtype=t.int16, device=self.dev)
        _check(lib().lgx_q8_repack_t16(self.handle, qs_rowmajor.data_ptr(), d_rowmajor.data_ptr(),
                                       n, k, out.data_ptr(), dout.data_ptr(), self._s()))
        return out, dout

    def unpack_t16(self, qs_t16, d_s16, n: int, k: int):
        t = self.torch
        out = t.empty((n, k), dtype=t.int8, device=self.dev)
        dout = t.empty((n, k // 32), dtype=t.int16, device=self.dev)
        _check(lib().lgx_q8_unpack_t16(self.handle, qs_t16.data_ptr(), d_s16.data_ptr(), n, k,
                                       out.data_ptr(), dout.data_ptr(), self._s()))
        return out, dout

    def to_device(self, a, dtype=None):
        """numpy array or tensor -> contiguous device tensor (uint16 data is
        carried as int16 bit patterns)."""
        t = self.torch
        if not isinstance(a, t.Tensor):
            import numpy as np

            a = np.ascontiguousarray(a)
            if a.dtype == np.uint16:
                a = a.view(np.int16)
            a = t.from_numpy(a)
        elif a.dtype == t.uint16:
            a = a.view(t.int16)
        if dtype is not None and a.dtype != dtype:
            a = a.to(dtype)
        return a.to(self.dev).contiguous()

    def q8_matrix(self, qs_rowmajor, d) -> Q8Matrix:
        """Upload (if host) and repack row-major quants + binary16 scale bits."""
        t = self.torch
        qs = self.to_device(qs_rowmajor, t.int8)
        dd = self.to_device(d, t.int16)
        n, k = qs.shape
        qt, ds = self.repack_t16(qs, dd)
        return Q8Matrix(qt, ds, n, k)

    # ---- Q8_0 ------------------------------------------------------------
    def quantize_q8_0(self, x, qs=None, d=None):
        t = self.torch
        m, k = x.shape
        qs = t.empty((m, k), dtype=t.int8, device=self.dev) if qs is None else qs
        d = t.empty((m, k // 32), dtype=t.int16, device=self.dev) if d is None else d
        _check(lib().lgx_quantize_q8_0(self.handle, x.data_ptr(), m, k, qs.data_ptr(),
                                       d.data_ptr(), self._s()))
        return qs, d

    def q8_gemv_f32(self, W: Q8Matrix, x, y=None):
        y = self.torch.empty(W.n, dtype=self.torch.float32, device=self.dev) if y is None else y
        _check(lib().lgx_q8_gemv_f32(self.handle, W.cstruct, x.data_ptr(), y.data_ptr(),
                                     self._s()))
        return y

    def q8q8_gemv(self, W: Q8Matrix, xq, xd, y=None, blockdots: bool = False):
        t = self.torch
        y = t.empty(W.n, dtype=t.float32, device=self.dev) if y is None else y
        dbg = t.empty((W.n, W.k // 32), dtype=t.int32, device=self.dev) if blockdots else None
        _check(lib().lgx_q8q8_gemv(self.handle, W.cstruct, xq.data_ptr(), xd.data_ptr(),
                                   y.data_ptr(), dbg.data_ptr() if dbg is not None else None,
                                   self._s()))
        return (y, dbg) if blockdots else y

    def q8q8_gemv_quantize(self, W: Q8Matrix, x, y=None, xq_out=None, xd_out=None):
        """y = W Q8_0(x) with the quantisation fused into the GEMV."""
        t = self.torch
        y = t.empty(W.n, dtype=t.float32, device=self.dev) if y is None else y
        _check(lib().lgx_q8q8_gemv_quantize(
            self.handle, W.cstruct, x.data_ptr(), y.data_ptr(),
            xq_out.data_ptr() if xq_out is not None else None,
            xd_out.data_ptr() if xd_out is not None else None, self._s()))
        return y

    def q8q8_gemv_quantize_group(self, Ws, xs, ys=None):
        """ys[i] = Ws[i] Q8_0(xs[i]) for up to 8 matrices in one launch."""
        t = self.torch
        n = len(Ws)
        ys = [t.empty(W.n, dtype=t.float32, device=self.dev) for W in Ws] if ys is None else ys
        arr = (Q8MatrixC * n)(*[W._c for W in Ws])
        xp = (C.c_void_p * n)(*[x.data_ptr() for x in xs])
        yp = (C.c_void_p * n)(*[y.data_ptr() for y in ys])
        _check(lib().lgx_q8q8_gemv_quantize_group(self.handle, n, arr, xp, yp, self._s()))
        return ys

    def q8_gemm_quantize_group(self, Ws, xs, ys=None):
        """ys[i] = Q8_0(xs[i]) Ws[i]^T for up to 8 matrices (xs[i]: [m][k_i]
        binary32, the same m for all) in three launches."""
        t = self.torch
        n = len(Ws)
        m = xs[0].shape[0] if xs[0].dim() == 2 else 1
        for x, W in zip(xs, Ws):
            if (x.shape[0] if x.dim() == 2 else 1) != m or x.shape[-1] != W.k or not x.is_contiguous():
                raise ValueError("every x must be a contiguous [m][k] of its matrix")
        ys = [t.empty((m, W.n), dtype=t.float32, device=self.dev) for W in Ws] if ys is None else ys
        arr = (Q8MatrixC * n)(*[W._c for W in Ws])
        xp = (C.c_void_p * n)(*[x.data_ptr() for x in xs])
        yp = (C.c_void_p * n)(*[y.data_ptr() for y in ys])
        _check(lib().lgx_q8_gemm_quantize_group(self.handle, n, arr, xp, m, yp, self._s()))
        return ys

    def q8q8_gemv_quantize_partials(self, W: Q8Matrix, x, part=None):
        t = self.torch
        g = lib().lgx_q8_range_count(W.k)
        part = t.empty((g, W.n), dtype=t.float32, device=self.dev) if part is None else part
        _check(lib().lgx_q8q8_gemv_quantize_partials(self.handle, W.cstruct, x.data_ptr(),
                                                     part.data_ptr(), None, None, self._s()))
        return part

    def q8_gemm_partials(self, W: Q8Matrix, xq, xd, part=None):
        t = self.torch
        m = xq.shape[0] if xq.dim() == 2 else 1
        g = lib().lgx_q8_range_count(W.k)
        part = t.empty((g, m, W.n), dtype=t.float32, device=self.dev) if part is None else part
        _check(lib().lgx_q8_gemm_partials(self.handle, W.cstruct, xq.data_ptr(), xd.data_ptr(), m,
                                          part.data_ptr(), self._s()))
        return part

    def range_combine(self, part, y=None):
        t = self.torch
        g = part.shape[0]
        count = part[0].numel()
        y = t.empty(part.shape[1:], dtype=t.float32, device=self.dev) if y is None else y
        _check(lib().lgx_q8_range_combine(self.handle, part.data_ptr(), g, count, y.data_ptr(),
                                          self._s()))
        return y

    def gqa_decode_attn(self, q, kpages, vpages, page_table, seq_len, max_seq_len: int,
                        out=None):
        """q [B][hq][d] f32; pages [P][hkv][16][d] (int16 bit patterns of binary16)."""
        t = self.torch
        B, hq, d = q.shape
        num_pages, hkv = kpages.shape[0], kpages.shape[1]
        maxp = page_table.shape[1]
        out = t.empty((B, hq, d), dtype=t.float32, device=self.dev) if out is None else out
        _check(lib().lgx_gqa_decode_attn(self.handle, q.data_ptr(), kpages.data_ptr(),
                                         vpages.data_ptr(), page_table.data_ptr(),
                                         seq_len.data_ptr(), B, hq, hkv, d, maxp, num_pages,
                                         max_seq_len, out.data_ptr(), self._s()))
        return out

    def gqa_prefill_attn(self, q, kpages, vpages, page_table, seq_len, P: int, max_seq_len: int,
                         out=None, fast: bool = False):
        """q [B*P][hq][d] f32: row b*P + j is the query at position seq_len[b] + j
        (causal over the first seq_len[b] + j + 1 cached tokens).  fast: the
        binary16 MFMA flash attention (within 2e-3 of the canonical result)."""
        t = self.torch
        rows, hq, d = q.shape
        B = seq_len.numel()
        if rows != B * P:
            raise ValueError(f"q has {rows} rows, expected B*P = {B * P}")
        num_pages, hkv = kpages.shape[0], kpages.shape[1]
        maxp = page_table.shape[1]
        out = t.empty((rows, hq, d), dtype=t.float32, device=self.dev) if out is None else out
        fn = lib().lgx_gqa_prefill_attn_fast if fast else lib().lgx_gqa_prefill_attn
        _check(fn(self.handle, q.data_ptr(), kpages.data_ptr(), vpages.data_ptr(),
                  page_table.data_ptr(), seq_len.data_ptr(), B, P, hq, hkv, d, maxp, num_pages,
                  max_seq_len, out.data_ptr(), self._s()))
        return out

    # ---- 8-bit KV cache --------------------------------------------------
    def rope_kv_append_i8(self, qkv, bias, rope: Rope, seq_len, page_table, kv: KvCacheI8, P: int = 1,
                          n_new=None, q_out=None):
        """Rotates and appends rows [B*P][(hq + 2 hkv) d] (row b*P + j: token
        seq_len[b] + j, j < n_new[b]) to the cache; returns the rotated queries
        [B*P][hq][d]."""
        t = self.torch
        B, maxp = page_table.shape
        d, hkv = kv.d, kv.hkv
        rows, width = qkv.shape
        hq = width // d - 2 * hkv
        if rows != B * P or hq < 1 or width % d:
            raise ValueError(f"qkv {tuple(qkv.shape)} is not [{B * P}][(hq + {2 * hkv}) * {d}]")
        _tensor("qkv", qkv, t.float32, qkv.shape, self.dev)
        if bias is not None:
            _tensor("bias", bias, t.float32, (width,), self.dev)
        if rope.device != self.dev:
            raise ValueError(f"the rotation's tables are on {rope.device}, the context on {self.dev}")
        self._lengths(seq_len, n_new, page_table, kv, B)
        q_out = t.empty((rows, hq, d), dtype=t.float32, device=self.dev) if q_out is None else \
            _tensor("q_out", q_out, t.float32, (rows, hq, d), self.dev)
        _check(lib().lgx_rope_kv_append_i8(
            self.handle, qkv.data_ptr(), _ptr_or_none(bias), rope.cstruct, seq_len.data_ptr(),
            _ptr_or_none(n_new), page_table.data_ptr(), kv.cstruct, q_out.data_ptr(), B, P, hq, maxp, self._s()))
        return q_out

    def kv_read_i8(self, kv: KvCacheI8, page_table, start, n: int, k_out=None, v_out=None):
        """(K, V) of tokens start[b] .. + n of every sequence, float32 [B][n][hkv][d]."""
        t = self.torch
        B, maxp = page_table.shape
        self._lengths(start, None, page_table, kv, B)
        shape = (B, n, kv.hkv, kv.d)
        k_out = t.empty(shape, dtype=t.float32, device=self.dev) if k_out is None else \
            _tensor("k_out", k_out, t.float32, shape, self.dev)
        v_out = t.empty(shape, dtype=t.float32, device=self.dev) if v_out is None else \
            _tensor("v_out", v_out, t.float32, shape, self.dev)
        _check(lib().lgx_kv_read_i8(self.handle, kv.cstruct, page_table.data_ptr(), start.data_ptr(), B, n, maxp,
                                    k_out.data_ptr(), v_out.data_ptr(), self._s()))
        return k_out, v_out

    def _lengths(self, seq_len, n_new, page_table, kv, B):
        if kv.device != self.dev:
            raise ValueError(f"the cache is on {kv.device}, the context on {self.dev}")
        i32 = self.torch.int32
        _tensor("page_table", page_table, i32, (B, page_table.shape[-1]), self.dev)
        _tensor("lengths", seq_len, i32, (B,), self.dev)
        if n_new is not None:
            _tensor("n_new", n_new, i32, (B,), self.dev)

    def gqa_decode_attn_i8(self, q, kv: KvCacheI8, page_table, seq_len, max_seq_len: int, opts: AttnOpts = None,
                           out=None):
        """q [B][hq][d] over the first seq_len[b] tokens of the 8-bit cache."""
        B, hq, d = q.shape
        if d != kv.d or page_table.shape[:1] != (B,):
            raise ValueError(f"q {tuple(q.shape)} for heads of {kv.d} and a page table {tuple(page_table.shape)}")
        self._lengths(seq_len, None, page_table, kv, B)
        out = self._attn_out(q, opts, out)
        _check(lib().lgx_gqa_decode_attn_i8(
            self.handle, q.data_ptr(), kv.cstruct, page_table.data_ptr(), seq_len.data_ptr(), B, hq,
            page_table.shape[1], max_seq_len, opts.cstruct if opts is not None else None, out.data_ptr(), self._s()))
        return out

    def gqa_prefill_attn_i8(self, q, kv: KvCacheI8, page_table, seq_len, P: int, max_seq_len: int, n_new=None,
                            opts: AttnOpts = None, out=None):
        """q [B*P][hq][d]: row b*P + j (j < n_new[b]) is the query at position
        seq_len[b] + j, causal over the 8-bit cache."""
        (B, _), (rows, hq, d) = page_table.shape, q.shape
        if rows != B * P or d != kv.d:
            raise ValueError(f"q {tuple(q.shape)} is not [{B * P}][hq][{kv.d}]")
        self._lengths(seq_len, n_new, page_table, kv, B)
        out = self._attn_out(q, opts, out)
        _check(lib().lgx_gqa_prefill_attn_i8(
            self.handle, q.data_ptr(), kv.cstruct, page_table.data_ptr(), seq_len.data_ptr(), _ptr_or_none(n_new),
            B, P, hq, page_table.shape[1], max_seq_len, opts.cstruct if opts is not None else None, out.data_ptr(),
            self._s()))
        return out

    def _attn_out(self, q, opts, out):
        f32 = self.torch.float32
        _tensor("q", q, f32, q.shape, self.dev)
        if opts is not None and opts.slopes is not None:
            _tensor("slopes", opts.slopes, f32, (q.shape[1],), self.dev)
        if out is None:
            return self.torch.empty_like(q)
        return _tensor("out", out, f32, q.shape, self.dev)

    # ---- drafted tokens --------------------------------------------------
    def tree_plan(self, parent, n_nodes=None):
        """(depth [B][N] int32, mask [B][N][ceil(N / 64)] int64) of trees of drafts given by
        every node's parent [B][N] (-1: hangs from the cached tokens)."""
        t = self.torch
        _tensor("parent", parent, t.int32, (None, None), self.dev)
        B, N = parent.shape
        if n_nodes is not None:
            _tensor("n_nodes", n_nodes, t.int32, (B,), self.dev)
        depth = t.zeros((B, N), dtype=t.int32, device=self.dev)
        mask = t.zeros((B, N, (N + 63) // 64), dtype=t.int64, device=self.dev)
        _check(lib().lgx_tree_plan(self.handle, parent.data_ptr(), _ptr_or_none(n_nodes), B, N, depth.data_ptr(),
                                   mask.data_ptr(), self._s()))
        return depth, mask

    def rope_kv_append_rows(self, qkv, bias, rope: Rope, seq_len, page_table, kv: KvCacheF16, N: int = 1, depth=None,
                            n_new=None, q_out=None):
        """Rotates and appends rows [B*N][(hq + 2 hkv) d] (row b*N + j: slot seq_len[b] + j,
        position seq_len[b] + depth[b][j], or + j) to the binary16 cache; returns the rotated
        queries [B*N][hq][d].  Rows of padding (n_new) are q_out's own; without q_out they
        hold anything."""
        t = self.torch
        B, maxp = page_table.shape
        d, hkv = kv.d, kv.hkv
        rows, width = qkv.shape
        hq = width // d - 2 * hkv
        if rows != B * N or hq < 1 or width % d:
            raise ValueError(f"qkv {tuple(qkv.shape)} is not [{B * N}][(hq + {2 * hkv}) * {d}]")
        _tensor("qkv", qkv, t.float32, qkv.shape, self.dev)
        if bias is not None:
            _tensor("bias", bias, t.float32, (width,), self.dev)
        if rope.device != self.dev:
            raise ValueError(f"the rotation's tables are on {rope.device}, the context on {self.dev}")
        self._lengths(seq_len, n_new, page_table, kv, B)
        if depth is not None:
            _tensor("depth", depth, t.int32, (B, N), self.dev)
        q_out = t.empty((rows, hq, d), dtype=t.float32, device=self.dev) if q_out is None else \
            _tensor("q_out", q_out, t.float32, (rows, hq, d), self.dev)
        _check(lib().lgx_rope_kv_append_rows(
            self.handle, qkv.data_ptr(), _ptr_or_none(bias), rope.cstruct, seq_len.data_ptr(), _ptr_or_none(depth),
            _ptr_or_none(n_new), page_table.data_ptr(), kv.cstruct, q_out.data_ptr(), B, N, hq, maxp, self._s()))
        return q_out

    def gqa_tree_attn(self, q, kv: KvCacheF16, page_table, seq_len, N: int, max_seq_len: int, mask=None, depth=None,
                      n_nodes=None, opts: AttnOpts = None, out=None):
        """q [B*N][hq][d]: row b*N + j is node j of sequence b, whose keys and values are
        in slot seq_len[b] + j of the binary16 cache; it sees the first seq_len[b] tokens
        and the nodes of mask [B][N][ceil(N / 64)] (int64 words; None: nodes 0 .. j).  Rows of
        padding (n_nodes) are out's own; without out they hold anything."""
        t = self.torch
        (B, maxp), (rows, hq, d) = page_table.shape, q.shape
        if rows != B * N or d != kv.d:
            raise ValueError(f"q {tuple(q.shape)} is not [{B * N}][hq][{kv.d}]")
        self._lengths(seq_len, n_nodes, page_table, kv, B)
        if mask is not None:
            _tensor("mask", mask, t.int64, (B, N, (N + 63) // 64), self.dev)
        if depth is not None:
            _tensor("depth", depth, t.int32, (B, N), self.dev)
        out = self._attn_out(q, opts, out)
        _check(lib().lgx_gqa_tree_attn(
            self.handle, q.data_ptr(), kv.cstruct, page_table.data_ptr(), seq_len.data_ptr(), _ptr_or_none(n_nodes),
            _ptr_or_none(depth), _ptr_or_none(mask), B, N, hq, maxp, max_seq_len,
            opts.cstruct if opts is not None else None, out.data_ptr(), self._s()))
        return out

    def tree_accept(self, tokens, parent, picked, seq_len=None, n_nodes=None, next_tokens=None):
        """(path [B][N], count [B], next token [B], seq_len + count or None): the nodes from
        node 0 on whose tokens were picked behind their parents."""
        t = self.torch
        i32, dev = t.int32, self.dev
        if tokens.dim() != 2:
            raise ValueError(f"tokens {tuple(tokens.shape)} is not [sequences][nodes]")
        B, N = shape = tokens.shape
        _tensor("tokens", tokens, i32, shape, dev)
        _tensor("parent", parent, i32, shape, dev)
        _tensor("picked", picked, i32, shape, dev)
        for name, x in (("seq_len", seq_len), ("n_nodes", n_nodes), ("next_tokens", next_tokens)):
            if x is not None:
                _tensor(name, x, i32, (B,), dev)
        path = t.empty(shape, dtype=i32, device=dev)
        count = t.empty(B, dtype=i32, device=dev)
        if next_tokens is None:
            next_tokens = (t.empty if n_nodes is None else t.zeros)(B, dtype=i32, device=dev)
        lens = t.empty(B, dtype=i32, device=dev) if seq_len is not None else None
        _check(lib().lgx_tree_accept(self.handle, tokens.data_ptr(), parent.data_ptr(), picked.data_ptr(),
                                     _ptr_or_none(n_nodes), _ptr_or_none(seq_len), B, N, path.data_ptr(), count.data_ptr(),
                                     next_tokens.data_ptr(), _ptr_or_none(lens), self._s()))
        return path, count, next_tokens, lens

    def kv_keep(self, caches, page_table, start, keep, n_keep) -> None:
        """Rows start[b] + keep[b][i], i < n_keep[b], become rows start[b] + i in every cache
        (a list of KvCacheF16, one per layer)."""
        t = self.torch
        caches = list(caches)
        if not caches:
            raise ValueError("no caches")
        if keep.dim() != 2:
            raise ValueError(f"keep {tuple(keep.shape)} is not [sequences][rows]")
        B, N = keep.shape
        _tensor("keep", keep, t.int32, (page_table.shape[0], N), self.dev)
        # dozens of layers: strings compare in a fifth of the time of torch's devices
        if {kv.where for kv in caches} != {self.where}:
            raise ValueError(f"caches on {sorted({kv.where for kv in caches})}, the context on {self.dev}")
        self._lengths(start, n_keep, page_table, caches[0], B)
        array = (KvF16C * len(caches)).from_buffer_copy(b"".join([kv.raw for kv in caches]))
        _check(lib().lgx_kv_keep(self.handle, array, len(caches), page_table.data_ptr(), start.data_ptr(), keep.data_ptr(),
                                 n_keep.data_ptr(), B, N, page_table.shape[1], self._s()))

    def sample_filtered(self, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, out=None, prob=None):
        """(tokens [m] int32, their probabilities [m]) of rows of logits [m][vocab] (a row
        may be longer in memory) by given random numbers u [m] of [0, 1) and per-row settings:
        float32 [m] temperature, top_p, min_p, int32 [m] top_k."""
        t = self.torch
        if logits.dim() != 2 or logits.dtype is not t.float32 or logits.device != self.dev or \
                (logits.shape[1] > 1 and logits.stride(1) != 1):
            raise ValueError(f"logits must be float32 rows [m][vocab] on {self.dev}, not {logits.dtype} {tuple(logits.shape)} "
                             f"on {logits.device}")
        m, vocab = logits.shape
        for name, x, dtype in (("u", u, t.float32), ("temperature", temperature, t.float32), ("top_k", top_k, t.int32),
                               ("top_p", top_p, t.float32), ("min_p", min_p, t.float32)):
            if x is not None or name == "u":
                _tensor(name, x, dtype, (m,), self.dev)
        out = t.empty(m, dtype=t.int32, device=self.dev) if out is None else _tensor("out", out, t.int32, (m,), self.dev)
        prob = t.empty(m, dtype=t.float32, device=self.dev) if prob is None else \
            _tensor("prob", prob, t.float32, (m,), self.dev)
        _check(lib().lgx_sample_filtered(
            self.handle, logits.data_ptr(), logits.stride(0) if m > 1 else vocab, m, vocab, _ptr_or_none(temperature),
            _ptr_or_none(top_k), _ptr_or_none(top_p), _ptr_or_none(min_p), u.data_ptr(), out.data_ptr(), prob.data_ptr(),
            self._s()))
        return out, prob

    # ---- pages of a cache ------------------------------------------------
    def _pool(self, pool, page_table, **lengths):
        dev, i32 = self.dev, self.torch.int32
        if pool.device != dev:
            raise ValueError(f"the pool is on {pool.device}, the context on {dev}")
        if page_table.dim() != 2:
            raise ValueError(f"page_table {tuple(page_table.shape)} is not [sequences][pages]")
        shape = page_table.shape
        _tensor("page_table", page_table, i32, shape, dev)
        for name, x in lengths.items():
            _tensor(name, x, i32, shape[:1], dev)
        return shape

    def pages_fork(self, pool: PagePool, page_table, seq_len, src, dst) -> None:
        """Sequence dst[i] becomes a copy of sequence src[i], sharing its pages."""
        S, maxp = self._pool(pool, page_table, seq_len=seq_len)
        i32, n = self.torch.int32, src.numel()
        _tensor("src", src, i32, (n,), self.dev)
        _tensor("dst", dst, i32, (n,), self.dev)
        _check(lib().lgx_pages_fork(self.handle, pool.cstruct, page_table.data_ptr(), seq_len.data_ptr(), src.data_ptr(),
                                    dst.data_ptr(), S, n, maxp, self._s()))

    def pages_reserve(self, pool: PagePool, page_table, seq_len, need, out=None):
        """Room for need[b] tokens behind seq_len[b]: (copies [B][2], n_copies [1],
        lacking [1]); the copies are pages_copy's.  If lacking[0] is not 0 no sequence
        got room, and none may be appended to."""
        B, maxp = self._pool(pool, page_table, seq_len=seq_len, need=need)
        t = self.torch
        shapes = ((B, 2), (1,), (1,))
        if out is None:
            out = tuple(t.zeros(s, dtype=t.int32, device=self.dev) for s in shapes)
        for name, x, s in zip(("copies", "n_copies", "lacking"), out, shapes, strict=True):
            _tensor(name, x, t.int32, s, self.dev)
        _check(lib().lgx_pages_reserve(self.handle, pool.cstruct, page_table.data_ptr(), seq_len.data_ptr(), need.data_ptr(),
                                       B, maxp, *(x.data_ptr() for x in out), self._s()))
        return out

    def pages_copy(self, planes: PagePlanes, copies, n_copies) -> None:
        """Copies page copies[i][0] to copies[i][1], i < n_copies[0], in every plane."""
        if planes.device != self.dev:
            raise ValueError(f"the planes are on {planes.device}, the context on {self.dev}")
        i32, n = self.torch.int32, copies.numel() // 2
        _tensor("copies", copies, i32, (n, 2), self.dev)
        _tensor("n_copies", n_copies, i32, (1,), self.dev)
        _check(lib().lgx_pages_copy(self.handle, planes.carray, planes.count, planes.num_pages, copies.data_ptr(),
                                    n_copies.data_ptr(), n, self._s()))

    def pages_free(self, pool: PagePool, page_table, keep) -> None:
        """Gives back the pages past each sequence's first keep[b] tokens."""
        B, maxp = self._pool(pool, page_table, keep=keep)
        _check(lib().lgx_pages_free(self.handle, pool.cstruct, page_table.data_ptr(), keep.data_ptr(), B, maxp, self._s()))

    def q8_gemm(self, W: Q8Matrix, xq, xd, y=None):
        t = self.torch
        m = xq.shape[0]
        y = t.empty((m, W.n), dtype=t.float32, device=self.dev) if y is None else y
        _check(lib().lgx_q8_gemm(self.handle, W.cstruct, xq.data_ptr(), xd.data_ptr(), m,
                                 y.data_ptr(), self._s()))
        return y

    def q8_gemm_noalloc(self, W: Q8Matrix, xq, xd, y):
        """lgx_q8_gemm_noalloc: the same product into the caller's y, with the
        library's fixed device scratch instead of any allocation."""
        m = xq.shape[0]
        _check(lib().lgx_q8_gemm_noalloc(self.handle, W.cstruct, xq.data_ptr(), xd.data_ptr(), m,
                                         y.data_ptr(), self._s()))
        return y

    # ---- decode-step glue ------------------------------------------------
    def embed_f16(self, emb, tokens, out=None):
        t = self.torch
        vocab, h = emb.shape
        m = tokens.numel()
        out = t.empty((m, h), dtype=t.float32, device=self.dev) if out is None else out
        _check(lib().lgx_embed_f16(self.handle, emb.data_ptr(), tokens.data_ptr(), m, h, vocab,
                                   out.data_ptr(), self._s()))
        return out

    def rmsnorm_quant(self, x, w, eps: float, y: bool = True, q8: bool = True):
        """(y, xq, xd) of RMSNorm(x) * w; unrequested outputs are None."""
        t = self.torch
        m, n = x.shape
        yo = t.empty((m, n), dtype=t.float32, device=self.dev) if y else None
        xq = t.empty((m, n), dtype=t.int8, device=self.dev) if q8 else None
        xd = t.empty((m, n // 32), dtype=t.int16, device=self.dev) if q8 else None
        _check(lib().lgx_rmsnorm_quant(self.handle, x.data_ptr(), w.data_ptr(), m, n, eps,
                                       _ptr_or_none(yo), _ptr_or_none(xq), _ptr_or_none(xd),
                                       self._s()))
        return yo, xq, xd

    def add_rmsnorm_quant(self, part, h, w, eps: float, y: bool = True, q8: bool = True):
        """h += tree(part) in place; then (y, xq, xd) of RMSNorm(h) * w."""
        t = self.torch
        nr, m, n = part.shape
        yo = t.empty((m, n), dtype=t.float32, device=self.dev) if y else None
        xq = t.empty((m, n), dtype=t.int8, device=self.dev) if q8 else None
        xd = t.empty((m, n // 32), dtype=t.int16, device=self.dev) if q8 else None
        _check(lib().lgx_add_rmsnorm_quant(self.handle, part.data_ptr(), nr, h.data_ptr(),
                                           w.data_ptr(), m, n, eps, _ptr_or_none(yo),
                                           _ptr_or_none(xq), _ptr_or_none(xd), self._s()))
        return yo, xq, xd

    def rope_kv_append(self, qkv, bias, cos_t, sin_t, seq_len, page_table, kpages, vpages,
                       hq: int, max_seq: int, q_out=None):
        t = self.torch
        B = qkv.shape[0]
        num_pages, hkv, _, d = kpages.shape
        maxp = page_table.shape[1]
        q_out = t.empty((B, hq, d), dtype=t.float32, device=self.dev) if q_out is None else q_out
        _check(lib().lgx_rope_kv_append(
            self.handle, qkv.data_ptr(), _ptr_or_none(bias), cos_t.data_ptr(), sin_t.data_ptr(),
            seq_len.data_ptr(), page_table.data_ptr(), kpages.data_ptr(), vpages.data_ptr(),
            q_out.data_ptr(), B, hq, hkv, d, maxp, num_pages, max_seq, self._s()))
        return q_out

    def swiglu_quant(self, gu, y: bool = True, q8: bool = True):
        t = self.torch
        m, i2 = gu.shape
        inter = i2 // 2
        yo = t.empty((m, inter), dtype=t.float32, device=self.dev) if y else None
        xq = t.empty((m, inter), dtype=t.int8, device=self.dev) if q8 else None
        xd = t.empty((m, inter // 32), dtype=t.int16, device=self.dev) if q8 else None
        _check(lib().lgx_swiglu_quant(self.handle, gu.data_ptr(), m, inter, _ptr_or_none(yo),
                                      _ptr_or_none(xq), _ptr_or_none(xd), self._s()))
        return yo, xq, xd

    def lm_head_f16(self, x, emb, out=None):
        t = self.torch
        m, h = x.shape
        vocab = emb.shape[0]
        out = t.empty((m, vocab), dtype=t.float32, device=self.dev) if out is None else out
        _check(lib().lgx_lm_head_f16(self.handle, x.data_ptr(), emb.data_ptr(), m, h, vocab,
                                     out.data_ptr(), self._s()))
        return out

    def f16_repack_t64(self, emb):
        """binary16 rows (int16/uint16 bits, [rows][h]) -> T64 order (flat)."""
        t = self.torch
        rows, h = emb.shape
        out = t.empty(int(lib().lgx_f16_t64_count(rows, h)), dtype=t.int16, device=self.dev)
        _check(lib().lgx_f16_repack_t64(self.handle, emb.data_ptr(), rows, h, out.data_ptr(),
                                        self._s()))
        return out

    def lm_head_f16_t64(self, x, emb_t64, vocab, out=None):
        t = self.torch
        m, h = x.shape
        out = t.empty((m, vocab), dtype=t.float32, device=self.dev) if out is None else out
        _check(lib().lgx_lm_head_f16_t64(self.handle, x.data_ptr(), emb_t64.data_ptr(), m, h,
                                         vocab, out.data_ptr(), self._s()))
        return out

    def lm_head_rowconst(self, emb):
        """Per-row constants of a binary16 embedding (int16 bits [vocab][h]) for
        lm_head_argmax_f16: float32 [vocab][4]."""
        t = self.torch
        vocab, h = emb.shape
        out = t.empty((vocab, 4), dtype=t.float32, device=self.dev)
        _check(lib().lgx_lm_head_rowconst(self.handle, emb.data_ptr(), vocab, h, out.data_ptr(),
                                          self._s()))
        return out

    def lm_head_argmax_f16(self, x, emb, emb_t64, rowc, out=None, bounds: bool = False):
        """Certified greedy token of the tied lm_head (the token of
        argmax(lm_head_f16(x, emb))); with bounds=True also the [m][vocab][2]
        scaled approximations and their bounds."""
        t = self.torch
        m, h = x.shape
        vocab = emb.shape[0]
        out = t.empty(m, dtype=t.int32, device=self.dev) if out is None else out
        bd = t.empty((m, vocab, 2), dtype=t.float32, device=self.dev) if bounds else None
        _check(lib().lgx_lm_head_argmax_f16(self.handle, x.data_ptr(), emb.data_ptr(),
                                            emb_t64.data_ptr(), rowc.data_ptr(), m, h, vocab,
                                            out.data_ptr(), bd.data_ptr() if bd is not None else None,
                                            self._s()))
        return (out, bd) if bounds else out

    def argmax(self, logits, out=None):
        t = self.torch
        m, vocab = logits.shape
        out = t.empty(m, dtype=t.int32, device=self.dev) if out is None else out
        _check(lib().lgx_argmax(self.handle, logits.data_ptr(), m, vocab, out.data_ptr(),
                                self._s()))
        return out

    def sample(self, logits, positions, top_k: int, top_p: float, temperature: float, seed: int,
               out=None):
        """lgx_sample: seeded top-k / top-p draw per row of logits [m][vocab];
        positions (device int32 [m]) are the draw indices of the rows' streams."""
        t = self.torch
        m, vocab = logits.shape
        out = t.empty(m, dtype=t.int32, device=self.dev) if out is None else out
        _check(lib().lgx_sample(self.handle, logits.data_ptr(), m, vocab, top_k, top_p,
                                temperature, seed, positions.data_ptr(), out.data_ptr(),
                                self._s()))
        return out


def _ptr_or_none(tensor):
    return tensor.data_ptr() if tensor is not None else None


class Model:
    """lgx_model: the seeded random-init Qwen2-shaped Q8_0 model on one device.

    ``cfg`` uses the oracle's keys (n_layers, hidden, inter, n_heads, n_kv,
    head_dim, vocab, tied, max_batch, max_seq, eps, theta, emb_sigma)."""

    def __init__(self, ctx: Context, cfg: dict, seed: int, _handle=None):
        self.ctx = ctx
        self.cfg = dict(cfg)
        self.c = QwenConfigC(cfg["n_layers"], cfg["hidden"], cfg["inter"], cfg["n_heads"],
                             cfg["n_kv"], cfg["head_dim"], cfg["vocab"], cfg["tied"],
                             cfg["max_batch"], cfg["max_seq"], cfg["eps"], cfg["theta"],
                             cfg["emb_sigma"])
        if _handle is None:
            h = C.c_void_p()
            _check(lib().lgx_model_create(ctx.handle, C.byref(self.c), seed, C.byref(h)))
            _handle = h
        self.handle = _handle
        ctx._models.add(self)

    @classmethod
    def load_gguf(cls, ctx: Context, path: str, max_batch: int, max_seq: int) -> "Model":
        """lgx_model_load_gguf: the model of a Qwen2 Q8_0 GGUF file."""
        h = C.c_void_p()
        _check(lib().lgx_model_load_gguf(ctx.handle, path.encode(), max_batch, max_seq,
                                         C.byref(h)))
        c = QwenConfigC()
        _check(lib().lgx_model_config(h, C.byref(c)))
        return cls(ctx, _cfg_dict(c), 0, _handle=h)

    def close(self) -> None:
        if self.handle:
            _check(lib().lgx_model_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def reset(self) -> None:
        _check(lib().lgx_model_reset(self.handle, self.ctx._s()))

    def set_sampling(self, temperature: float, top_k: int = 1, top_p: float = 1.0,
                     seed: int = 0) -> None:
        """Seeded top-k / top-p token choice for later steps (temperature 0:
        greedy)."""
        _check(lib().lgx_model_set_sampling(self.handle, temperature, top_k, top_p, seed))

    def set_prefill_mode(self, fast: bool) -> None:
        """fast: later prefills run in binary16 (LGX_PREFILL_FAST: binary16
        GEMMs and flash attention, the last position exact); the call does the
        mode's one-time work (binary16 weights, GEMM plans) and synchronises.
        Otherwise the exact canonical schedule."""
        _check(lib().lgx_model_set_prefill_mode(self.handle, 1 if fast else 0))

    def decode_step(self, tokens) -> None:
        """tokens: device int32 [B], replaced in place by the next tokens."""
        _check(lib().lgx_qwen_decode_step(self.handle, tokens.numel(), tokens.data_ptr(),
                                          self.ctx._s()))

    def generate(self, tokens, nsteps: int, history=None) -> None:
        """nsteps decode steps replayed from a recorded HIP graph; tokens
        (device int32 [B]) ends as the last step's next tokens and history
        (device int32 [nsteps][B], optional) receives every step's."""
        _check(lib().lgx_qwen_generate(self.handle, tokens.numel(), tokens.data_ptr(), nsteps,
                                       0 if history is None else history.data_ptr(),
                                       self.ctx._s()))

    def prefill(self, prompt, next_tokens=None):
        """prompt: device int32 [B][P]; returns the device int32 [B] next tokens."""
        t = self.ctx.torch
        B, P = prompt.shape
        nxt = t.empty(B, dtype=t.int32, device=self.ctx.dev) if next_tokens is None else next_tokens
        _check(lib().lgx_qwen_prefill(self.handle, B, P, prompt.data_ptr(), nxt.data_ptr(),
                                      self.ctx._s()))
        return nxt

    def logits(self, B: int):
        t = self.ctx.torch
        out = t.empty((B, self.cfg["vocab"]), dtype=t.float32, device=self.ctx.dev)
        _check(lib().lgx_qwen_logits(self.handle, B, out.data_ptr(), self.ctx._s()))
        return out

    def tensor_ptr(self, name: str, layer: int = 0):
        """(device pointer, bytes) of a model tensor."""
        p, n = C.c_void_p(), C.c_size_t()
        _check(lib().lgx_model_tensor(self.handle, layer, MODEL_TENSORS[name], C.byref(p),
                                      C.byref(n)))
        return int(p.value or 0), int(n.value)

    def tensor_bytes(self, name: str, layer: int = 0):
        """Host copy (numpy uint8) of a model tensor's bytes."""
        import numpy as np

        t = self.ctx.torch
        p, n = self.tensor_ptr(name, layer)
        t.cuda.current_stream(self.ctx.dev).synchronize()
        out = np.empty(n, np.uint8)
        _check_hip(C.CDLL("libamdhip64.so").hipMemcpy(
            out.ctypes.data_as(C.c_void_p), C.c_void_p(p), C.c_size_t(n), 2))
        return out


    def kv_rows(self, layer: int, which: int, b: int, n: int, page_table=None):
        """Host copy of the first n cached K (which 0) or V (1) rows of
        sequence b at `layer`: binary16 [n][n_kv][head_dim] (gathered page by
        page through the model's page table)."""
        import numpy as np

        cfg = self.cfg
        hkv, d = cfg["n_kv"], cfg["head_dim"]
        maxp = -(-cfg["max_seq"] // 16)
        if page_table is None:
            page_table = self.tensor_bytes("page_table").view(np.int32).reshape(
                cfg["max_batch"], maxp)
        p, _ = self.tensor_ptr("k_pages" if which == 0 else "v_pages", layer)
        page_bytes = hkv * 16 * d * 2
        npg = -(-n // 16)
        buf = np.empty((npg, hkv, 16, d), np.uint16)
        hip = C.CDLL("libamdhip64.so")
        self.ctx.torch.cuda.current_stream(self.ctx.dev).synchronize()
        for i in range(npg):
            _check_hip(hip.hipMemcpy(buf[i].ctypes.data_as(C.c_void_p),
                                     C.c_void_p(p + int(page_table[b, i]) * page_bytes),
                                     C.c_size_t(page_bytes), 2))
        return np.ascontiguousarray(buf.transpose(0, 2, 1, 3).reshape(npg * 16, hkv, d)[:n])


def _cfg_dict(c) -> dict:
    return dict(n_layers=c.n_layers, hidden=c.hidden, inter=c.intermediate, n_heads=c.n_heads,
                n_kv=c.n_kv_heads, head_dim=c.head_dim, vocab=c.vocab, tied=c.tied_embedding,
                max_batch=c.max_batch, max_seq=c.max_seq, eps=c.rms_eps, theta=c.rope_theta,
                emb_sigma=c.emb_sigma)


def gguf_config(path: str, max_batch: int, max_seq: int) -> dict:
    """lgx_gguf_config: the model shape of a Qwen2 GGUF file (host only)."""
    c = QwenConfigC()
    _check(lib().lgx_gguf_config(path.encode(), max_batch, max_seq, C.byref(c)))
    return _cfg_dict(c)


def _check_hip(err: int) -> None:
    if err != 0:
        raise LgxError(10, f"hipMemcpy failed with hipError {err}")
