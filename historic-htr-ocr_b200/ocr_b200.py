"""ocr_b200 — Python host binding of libocrcuda.so (the C ABI in include/ocr_cuda.h).

It mirrors the reference engine's text-decode API (b-straub/historic-htr-ocr, app/crates/ocr-wgpu/src/text.rs):
    TextModel.load(ctx, path)            ≡ TextModel::load (text.rs:332-375)
    model.session(n_ctx, batch)          ≡ TextModel::session / session_for (text.rs:378-434)
    session.prefill(slot, ids, embd)     ≡ TextModel::prefill (text.rs:437-521), Input::Tokens / Input::Embeddings
    session.step(tokens)                 ≡ TextModel::step (text.rs:524-537)
    session.decode_gpu(slot, preset, history, on_token)  ≡ Choice::new + TextModel::decode_gpu (text.rs:185, 587-625)
    choose_gpu(ctx, d_logits, …)         ≡ ocr_decode::sampling::choose, greedy (sampling.rs:38-62)
Errors raise OcrError with the library's message (anyhow's text in the reference). The library must be built
(historic-htr-ocr_b200/build.py); importing this module without it raises — there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import os
from dataclasses import dataclass
from pathlib import Path
from typing import Callable, Optional, Sequence

import numpy as np

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "lib" / "libocrcuda.so"

# ---------------------------------------------------------------------------------------------------------------------
# the library
# ---------------------------------------------------------------------------------------------------------------------


class OcrError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


class TextCfg(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("n_layer", "dim", "n_head", "n_kv", "d_head", "n_ff", "n_vocab",
                                          "n_ctx_train")] + [("eps", C.c_float), ("rope_base", C.c_float)]


class VisionCfg(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("n_layer", "dim", "n_head", "n_ff", "patch", "merge", "image_size",
                                         "proj_dim")] + [("eps", C.c_float), ("rope_theta", C.c_float),
                                                         ("mean", C.c_float * 3), ("std", C.c_float * 3)]


class BakePlan(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("scaled_w", "scaled_h", "left", "top", "right", "bottom")]


class SamplerCfg(C.Structure):
    _fields_ = [("rp", C.c_float), ("window", C.c_int32), ("fp", C.c_float), ("max_new", C.c_int32)]


class KernelTime(C.Structure):
    _fields_ = [("name", C.c_char * 32), ("layer", C.c_int32), ("us", C.c_float), ("bytes", C.c_double)]


TOKEN_CB = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_int32)


class Page(C.Structure):
    _fields_ = [("id", C.c_int64), ("ids", C.c_void_p), ("embd", C.c_void_p), ("n_rows", C.c_int32),
                ("history", C.c_void_p), ("n_hist", C.c_int32), ("max_new", C.c_int32), ("ids_out", C.c_void_p),
                ("n_out", C.c_int32)]


class KvCacheC(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("type", "n_slot", "n_kv", "d_head", "n_rows", "window", "sinks", "ring")] + \
        [(n, C.c_void_p) for n in ("k", "v", "k_scale", "v_scale")]


class Rows(C.Structure):
    """ocr_rows: vectors of d_head consecutive elements, slot b, row t, head h at the given strides"""
    _fields_ = [("data", C.c_void_p), ("half", C.c_int32)] + \
        [(n, C.c_int64) for n in ("slot_stride", "row_stride", "head_stride")]


PAGE_CB = C.CFUNCTYPE(C.c_int, C.c_void_p, C.POINTER(Page))


class PageIO(C.Structure):
    _fields_ = [("user", C.c_void_p), ("next", PAGE_CB), ("done", PAGE_CB)]

_P = C.c_void_p
_SIGS = {
    "ocr_last_error": (C.c_char_p, []),
    "ocr_version": (C.c_char_p, []),
    "ocr_ctx_create": (C.c_int, [C.c_int, C.POINTER(_P)]),
    "ocr_ctx_destroy": (C.c_int, [_P]),
    "ocr_ctx_sync": (C.c_int, [_P]),
    "ocr_ctx_stream": (C.c_int, [_P, C.POINTER(_P)]),
    "ocr_ctx_memory": (C.c_int, [_P, C.POINTER(C.c_uint64), C.POINTER(C.c_uint64), C.POINTER(C.c_uint64)]),
    "ocr_model_load_gguf": (C.c_int, [_P, C.c_char_p, C.POINTER(_P)]),
    "ocr_model_load_gguf_memory": (C.c_int, [_P, _P, C.c_size_t, C.POINTER(_P)]),
    "ocr_model_synthetic": (C.c_int, [_P, C.POINTER(TextCfg), C.c_uint64, C.c_float, C.c_float, C.POINTER(_P)]),
    "ocr_model_config": (C.c_int, [_P, C.POINTER(TextCfg)]),
    "ocr_model_tensor_gguf": (C.c_int, [_P, C.c_int, C.c_int, _P, C.POINTER(C.c_size_t)]),
    "ocr_model_checksum": (C.c_int, [_P, C.POINTER(C.c_uint64)]),
    "ocr_model_destroy": (C.c_int, [_P]),
    "ocr_session_create": (C.c_int, [_P, C.c_int, C.c_int, C.POINTER(_P)]),
    "ocr_session_destroy": (C.c_int, [_P]),
    "ocr_session_n_past": (C.c_int, [_P, C.c_int, C.POINTER(C.c_int)]),
    "ocr_session_rewind": (C.c_int, [_P, C.c_int, C.c_int]),
    "ocr_session_kv": (C.c_int, [_P, C.c_int, C.c_int, C.c_int, C.c_int, _P, _P]),
    "ocr_prefill": (C.c_int, [_P, C.c_int, _P, _P, C.c_int, _P]),
    "ocr_step": (C.c_int, [_P, _P, _P]),
    "ocr_decode": (C.c_int, [_P, C.c_int, C.POINTER(SamplerCfg), _P, C.c_int, TOKEN_CB, _P, _P,
                             C.POINTER(C.c_int)]),
    "ocr_decode_batch": (C.c_int, [_P, C.POINTER(SamplerCfg), _P, C.c_int, _P]),
    "ocr_read_pages": (C.c_int, [_P, C.POINTER(SamplerCfg), C.c_int, C.POINTER(PageIO)]),
    "ocr_step_embd": (C.c_int, [_P, _P, _P, _P]),
    "ocr_profile_step": (C.c_int, [_P, _P, C.POINTER(KernelTime), C.c_int, C.POINTER(C.c_int)]),
    "ocr_timeline_step": (C.c_int, [_P, _P, C.c_int, C.POINTER(KernelTime), C.c_int, C.POINTER(C.c_int)]),
    "ocr_sample_logits": (C.c_int, [_P, _P, C.c_int, C.POINTER(SamplerCfg), _P, C.c_int, _P, _P, C.c_int, _P]),
    "ocr_bake_plan_for": (C.c_int, [C.c_int, C.c_int, C.c_int, C.c_int, C.POINTER(BakePlan)]),
    "ocr_vision_synthetic": (C.c_int, [_P, C.POINTER(VisionCfg), C.c_uint64, C.c_float, C.POINTER(_P)]),
    "ocr_vision_destroy": (C.c_int, [_P]),
    "ocr_vision_config": (C.c_int, [_P, C.POINTER(VisionCfg)]),
    "ocr_vision_encode": (C.c_int, [_P, _P, C.c_int, C.c_int, C.c_int, _P, C.c_size_t, C.POINTER(C.c_int),
                                    C.POINTER(C.c_int)]),
    "ocr_vision_encode_page": (C.c_int, [_P, _P, C.c_int, C.c_int, _P, C.c_size_t, C.POINTER(C.c_int)]),
    "ocr_image_bake": (C.c_int, [_P, _P, C.c_int, C.c_int, C.c_int, C.c_int, _P, C.c_size_t, C.POINTER(C.c_int),
                                 C.POINTER(C.c_int)]),
    "ocr_gguf_open": (C.c_int, [C.c_char_p, C.POINTER(_P)]),
    "ocr_gguf_open_memory": (C.c_int, [_P, C.c_size_t, C.POINTER(_P)]),
    "ocr_gguf_close": (C.c_int, [_P]),
    "ocr_gguf_header": (C.c_int, [_P, C.POINTER(C.c_uint32), C.POINTER(C.c_uint64), C.POINTER(C.c_uint64),
                                  C.POINTER(C.c_uint64)]),
    "ocr_gguf_get_u32": (C.c_int, [_P, C.c_char_p, C.POINTER(C.c_uint32)]),
    "ocr_gguf_get_f32": (C.c_int, [_P, C.c_char_p, C.POINTER(C.c_float)]),
    "ocr_gguf_get_str": (C.c_int, [_P, C.c_char_p, C.c_char_p, C.c_size_t]),
    "ocr_gguf_f32_array": (C.c_int, [_P, C.c_char_p, _P, C.c_size_t, C.POINTER(C.c_size_t)]),
    "ocr_gguf_tensor": (C.c_int, [_P, C.c_char_p, C.POINTER(C.c_int), C.POINTER(C.c_uint64 * 4),
                                  C.POINTER(C.c_int), C.POINTER(C.c_uint64)]),
    "ocr_gguf_to_f32": (C.c_int, [_P, C.c_char_p, _P, C.c_size_t, C.POINTER(C.c_size_t)]),
    "ocr_gguf_text_config": (C.c_int, [_P, C.POINTER(TextCfg)]),
    "ocr_gguf_vision_config": (C.c_int, [_P, C.POINTER(VisionCfg)]),
    "ocr_op_penalize": (C.c_int, [_P, _P, C.c_int, C.c_float, C.c_int, _P, C.c_int]),
    "ocr_q8_row_bytes": (C.c_int, [C.c_int]),
    "ocr_op_repack_q8_0": (C.c_int, [_P, _P, C.c_int, C.c_int, _P]),
    "ocr_op_matvec_q8_0": (C.c_int, [_P, _P, C.c_int, C.c_int, _P, _P, C.c_float, C.c_int, _P, C.c_int]),
    "ocr_op_lm_head_sample": (C.c_int, [_P, _P, C.c_int, C.c_int, _P, _P, C.c_float, C.c_float, C.c_int, _P, _P, _P,
                                        _P]),
    "ocr_op_lm_head_sample_noalloc": (C.c_int, [_P, _P, C.c_int, C.c_int, _P, _P, C.c_float, C.c_float, C.c_int, _P,
                                                _P, _P, _P]),
    "ocr_kv_cache_bytes": (C.c_int, [C.POINTER(KvCacheC), C.POINTER(C.c_size_t), C.POINTER(C.c_size_t)]),
    "ocr_session_kv_cache": (C.c_int, [_P, C.c_int, C.POINTER(KvCacheC)]),
    "ocr_op_kv_write": (C.c_int, [_P, C.POINTER(KvCacheC), C.POINTER(Rows), C.POINTER(Rows), C.c_int, _P, _P]),
    "ocr_op_kv_read": (C.c_int, [_P, C.POINTER(KvCacheC), C.POINTER(Rows), C.POINTER(Rows), C.c_int, _P, _P]),
    "ocr_op_attention_window": (C.c_int, [_P, C.POINTER(KvCacheC), C.POINTER(Rows), C.c_int, C.c_int, _P, _P, C.c_float,
                                          C.POINTER(Rows)]),
    "ocr_op_attention_tree": (C.c_int, [_P, C.POINTER(KvCacheC), C.POINTER(Rows), C.c_int, C.c_int, _P, _P, _P,
                                        C.c_float, C.POINTER(Rows)]),
    "ocr_op_kv_keep": (C.c_int, [_P, C.POINTER(KvCacheC), C.c_int, C.c_int, _P, _P, _P]),
    "ocr_op_wait_probe": (C.c_int, [_P, C.c_int, C.POINTER(C.c_int)]),
    "ocr_op_attention_full": (C.c_int, [_P, _P, C.c_int, C.c_int, C.c_int, _P, _P, C.c_int, C.c_int, C.c_float, _P,
                                        C.c_int]),
    "ocr_op_attention_decode": (C.c_int, [_P, _P, _P, _P, _P, _P, _P, C.c_int, C.c_int, C.c_int, C.c_int, C.c_float,
                                          _P]),
}

# every symbol include/ocr_cuda.h declares (tests check the library exports each)
EXPORTS = tuple(_SIGS)

_lib: Optional[C.CDLL] = None


def lib() -> C.CDLL:
    """The loaded libocrcuda.so; raises if it is not built (no fallback of any kind)."""
    global _lib
    if _lib is None:
        path = Path(os.environ.get("OCR_B200_LIB", LIB_PATH))
        if not path.exists():
            raise OcrError(-1, f"{path} is not built: run historic-htr-ocr_b200/build.py")
        L = C.CDLL(str(path))
        for name, (res, args) in _SIGS.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
    return _lib


def _check(rc: int) -> None:
    if rc != 0:
        raise OcrError(rc, lib().ocr_last_error().decode(errors="replace"))


def _ptr(a) -> Optional[int]:
    """host numpy array → address (None stays NULL); torch tensors → their data_ptr()"""
    if a is None:
        return None
    if isinstance(a, int):
        return a
    if hasattr(a, "data_ptr"):
        return a.data_ptr()
    return a.ctypes.data


# ---------------------------------------------------------------------------------------------------------------------
# presets (app/crates/ocr-decode/src/presets.rs:18-57) — greedy only on the device (text.rs:151-163)
# ---------------------------------------------------------------------------------------------------------------------
@dataclass
class Preset:
    name: str = "greedy_rp1.1"
    temperature: float = 0.0
    top_p: float = 1.0
    repetition_penalty: float = 1.1
    repetition_window: int = 20
    frequency_penalty: float = 0.0
    max_new_tokens: int = 7024

    def greedy(self) -> bool:
        return self.temperature == 0.0

    def sampler(self, max_new: Optional[int] = None) -> SamplerCfg:
        if not self.greedy():
            raise OcrError(1, f"preset '{self.name}': sampled (temperature > 0): the token is drawn on the CPU")
        return SamplerCfg(float(self.repetition_penalty), int(self.repetition_window), float(self.frequency_penalty),
                          int(max_new if max_new is not None else self.max_new_tokens))


# the shipped presets (app/presets.json)
PRESETS = {
    "greedy_rp1.1": Preset("greedy_rp1.1", 0.0, 1.0, 1.1, 20, 0.0, 7024),
    "greedy_rp1.1_fp0.1": Preset("greedy_rp1.1_fp0.1", 0.0, 1.0, 1.1, 20, 0.1, 7024),
}


# ---------------------------------------------------------------------------------------------------------------------
# context / model / session
# ---------------------------------------------------------------------------------------------------------------------
class Context:
    """One device, one stream (Gpu::create's role)."""

    def __init__(self, device: int = 0):
        h = C.c_void_p()
        _check(lib().ocr_ctx_create(device, C.byref(h)))
        self.h = h
        self.device = device

    def close(self) -> None:
        if self.h:
            lib().ocr_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def sync(self) -> None:
        _check(lib().ocr_ctx_sync(self.h))

    def stream(self) -> int:
        s = C.c_void_p()
        _check(lib().ocr_ctx_stream(self.h, C.byref(s)))
        return s.value or 0

    def memory(self) -> dict:
        w, kv, wk = C.c_uint64(), C.c_uint64(), C.c_uint64()
        _check(lib().ocr_ctx_memory(self.h, C.byref(w), C.byref(kv), C.byref(wk)))
        return {"weights": w.value, "kv_cache": kv.value, "work": wk.value}


@dataclass
class TextConfig:
    n_layer: int = 28
    dim: int = 1024
    n_head: int = 16
    n_kv: int = 8
    d_head: int = 128
    n_ff: int = 3072
    n_vocab: int = 151936
    n_ctx_train: int = 40960
    eps: float = 1e-6
    rope_base: float = 1e6

    def c(self) -> TextCfg:
        return TextCfg(self.n_layer, self.dim, self.n_head, self.n_kv, self.d_head, self.n_ff, self.n_vocab,
                       self.n_ctx_train, self.eps, self.rope_base)

    @staticmethod
    def from_c(c: TextCfg) -> "TextConfig":
        return TextConfig(c.n_layer, c.dim, c.n_head, c.n_kv, c.d_head, c.n_ff, c.n_vocab, c.n_ctx_train, c.eps,
                          c.rope_base)


# tensor kinds of a layer (ocr_model_tensor_gguf numbering), with their GGUF names
KINDS = ("attn_norm", "attn_q", "attn_k", "attn_v", "attn_output", "attn_q_norm", "attn_k_norm", "ffn_norm",
         "ffn_gate", "ffn_up", "ffn_down")


class TextModel:
    def __init__(self, ctx: Context, h: C.c_void_p):
        self.ctx, self.h = ctx, h
        c = TextCfg()
        _check(lib().ocr_model_config(h, C.byref(c)))
        self.cfg = TextConfig.from_c(c)

    @classmethod
    def load(cls, ctx: Context, path: str) -> "TextModel":
        h = C.c_void_p()
        _check(lib().ocr_model_load_gguf(ctx.h, str(path).encode(), C.byref(h)))
        return cls(ctx, h)

    @classmethod
    def from_bytes(cls, ctx: Context, data: bytes) -> "TextModel":
        buf = C.create_string_buffer(data, len(data))
        h = C.c_void_p()
        _check(lib().ocr_model_load_gguf_memory(ctx.h, buf, len(data), C.byref(h)))
        return cls(ctx, h)

    @classmethod
    def synthetic(cls, ctx: Context, cfg: TextConfig, seed: int, sigma_w: float = 0.02,
                  sigma_e: float = 0.02) -> "TextModel":
        h = C.c_void_p()
        c = cfg.c()
        _check(lib().ocr_model_synthetic(ctx.h, C.byref(c), C.c_uint64(seed), sigma_w, sigma_e, C.byref(h)))
        return cls(ctx, h)

    def close(self) -> None:
        if self.h:
            lib().ocr_model_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def tensor_gguf(self, layer: int, kind: int) -> bytes:
        n = C.c_size_t(0)
        _check(lib().ocr_model_tensor_gguf(self.h, layer, kind, None, C.byref(n)))
        buf = C.create_string_buffer(n.value)
        _check(lib().ocr_model_tensor_gguf(self.h, layer, kind, buf, C.byref(n)))
        return buf.raw[: n.value]

    def checksum(self) -> int:
        x = C.c_uint64()
        _check(lib().ocr_model_checksum(self.h, C.byref(x)))
        return x.value

    def session(self, n_ctx: int, batch: int = 1) -> "Session":
        h = C.c_void_p()
        _check(lib().ocr_session_create(self.h, n_ctx, batch, C.byref(h)))
        return Session(self, h, n_ctx, batch)


# ---------------------------------------------------------------------------------------------------------------------
# the vision encoder + projector (Vision, app/crates/ocr-wgpu/src/vision.rs:37-450) and the bake's plan
# ---------------------------------------------------------------------------------------------------------------------
@dataclass
class VisionConfig:
    """VisionConfig (vision.rs:37-88); the defaults are the LightOnOCR mmproj's shape (Pixtral ViT, 1540 px)"""
    n_layer: int = 24
    dim: int = 1024
    n_head: int = 16
    n_ff: int = 4096
    patch: int = 14
    merge: int = 2
    image_size: int = 1540
    proj_dim: int = 1024
    eps: float = 1e-5
    rope_theta: float = 10000.0
    mean: tuple = (0.48145466, 0.4578275, 0.40821073)
    std: tuple = (0.26862954, 0.26130258, 0.27577711)

    def c(self) -> VisionCfg:
        return VisionCfg(self.n_layer, self.dim, self.n_head, self.n_ff, self.patch, self.merge, self.image_size,
                         self.proj_dim, self.eps, self.rope_theta, (C.c_float * 3)(*self.mean),
                         (C.c_float * 3)(*self.std))

    def as_dict(self) -> dict:
        return dict(n_layer=self.n_layer, dim=self.dim, n_head=self.n_head, n_ff=self.n_ff, patch=self.patch,
                    merge=self.merge, image_size=self.image_size, proj_dim=self.proj_dim, eps=self.eps,
                    rope_theta=self.rope_theta, mean=list(self.mean), std=list(self.std))


def bake_plan(longest: int, grid: int, w0: int, h0: int) -> tuple:
    """imageops.rs plan(Bake { longest, grid }, w0, h0): (scaled_w, scaled_h, left, top, right, bottom)"""
    p = BakePlan()
    _check(lib().ocr_bake_plan_for(longest, grid, w0, h0, C.byref(p)))
    return (p.scaled_w, p.scaled_h, p.left, p.top, p.right, p.bottom)


def image_bake(ctx: Context, rgb: np.ndarray, longest: int = 1540, grid: int = 28) -> np.ndarray:
    """imageops::bake on the device: the Lanczos-3 resize when the plan scales, then the white pads"""
    rgb = np.ascontiguousarray(rgb, np.uint8)
    h0, w0 = rgb.shape[:2]
    sw, sh, left, top, right, bottom = bake_plan(longest, grid, w0, h0)
    out = np.empty((sh + top + bottom, sw + left + right, 3), np.uint8)
    fw, fh = C.c_int(), C.c_int()
    _check(lib().ocr_image_bake(ctx.h, _ptr(rgb), w0, h0, longest, grid, _ptr(out), out.nbytes, C.byref(fw),
                                C.byref(fh)))
    return out


class Vision:
    def __init__(self, ctx: Context, h: C.c_void_p):
        self.ctx, self.h = ctx, h
        c = VisionCfg()
        _check(lib().ocr_vision_config(h, C.byref(c)))
        self.cfg = VisionConfig(c.n_layer, c.dim, c.n_head, c.n_ff, c.patch, c.merge, c.image_size, c.proj_dim, c.eps,
                                c.rope_theta, tuple(c.mean), tuple(c.std))

    @classmethod
    def synthetic(cls, ctx: Context, cfg: VisionConfig, seed: int, sigma_w: float = 0.02) -> "Vision":
        h = C.c_void_p()
        c = cfg.c()
        _check(lib().ocr_vision_synthetic(ctx.h, C.byref(c), C.c_uint64(seed), sigma_w, C.byref(h)))
        return cls(ctx, h)

    def close(self) -> None:
        if self.h:
            lib().ocr_vision_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def encode(self, rgb, layers: int = -1, out=None, w: int = 0, h: int = 0) -> np.ndarray:
        """Vision::encode: a baked rgb image (uint8 [h][w][3] numpy, or a device pointer with w, h) → the embeddings
        [n_tokens][proj_dim] (layers < 0) or the residual [n_patches][dim] after `layers` encoder layers. `out` (a
        torch tensor on the device, or None for a new host array) receives the rows."""
        if not isinstance(rgb, int):
            rgb = np.ascontiguousarray(rgb, np.uint8)
            h, w = rgb.shape[:2]
        c = self.cfg
        n = (w // c.patch) * (h // c.patch)
        rows, width = (n, c.dim) if layers >= 0 else (n // (c.merge * c.merge), c.proj_dim)
        host = out is None
        if host:
            out = np.empty((rows, width), np.float32)
        cap = rows * width if host else out.numel()
        nr, rw = C.c_int(), C.c_int()
        _check(lib().ocr_vision_encode(self.h, _ptr(rgb), w, h, layers, _ptr(out), cap, C.byref(nr), C.byref(rw)))
        return out

    def encode_page(self, rgb: np.ndarray, out=None) -> np.ndarray:
        """the bake (white pads, no resize) and the encode in one call: rgb uint8 [h0][w0][3]"""
        rgb = np.ascontiguousarray(rgb, np.uint8)
        h0, w0 = rgb.shape[:2]
        c = self.cfg
        sw, sh, left, top, right, bottom = bake_plan(c.image_size, c.patch * c.merge, w0, h0)
        g = c.patch * c.merge
        rows = ((sw + left + right) // g) * ((sh + top + bottom) // g)
        host = out is None
        if host:
            out = np.empty((rows, c.proj_dim), np.float32)
        cap = rows * c.proj_dim if host else out.numel()
        nr = C.c_int()
        _check(lib().ocr_vision_encode_page(self.h, _ptr(rgb), w0, h0, _ptr(out), cap, C.byref(nr)))
        return out


class Session:
    def __init__(self, model: TextModel, h: C.c_void_p, n_ctx: int, batch: int):
        self.model, self.h, self.n_ctx, self.batch = model, h, n_ctx, batch

    def close(self) -> None:
        if self.h:
            lib().ocr_session_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def n_past(self, slot: int = 0) -> int:
        n = C.c_int()
        _check(lib().ocr_session_n_past(self.h, slot, C.byref(n)))
        return n.value

    def rewind(self, slot: int, n_past: int) -> None:
        _check(lib().ocr_session_rewind(self.h, slot, n_past))

    def kv(self, layer: int, slot: int, row0: int, n_rows: int) -> tuple[np.ndarray, np.ndarray]:
        """KV rows [row0, row0 + n_rows) of a layer and slot: (k, v) f16 bit patterns [n_rows][n_kv * 128]"""
        w = self.model.cfg.n_kv * 128
        k = np.empty((n_rows, w), np.uint16)
        v = np.empty((n_rows, w), np.uint16)
        _check(lib().ocr_session_kv(self.h, layer, slot, row0, n_rows, _ptr(k), _ptr(v)))
        return k, v

    def kv_cache(self, layer: int) -> "KvCache":
        """a layer's KV rows, live, as an f16 cache for the op_kv_* and op_attention_* calls"""
        c = KvCacheC()
        _check(lib().ocr_session_kv_cache(self.h, layer, C.byref(c)))
        return KvCache._of(c, self)

    def prefill(self, slot: int = 0, ids: Optional[Sequence[int]] = None, embd: Optional[np.ndarray] = None,
                logits: bool = True) -> Optional[np.ndarray]:
        """rows: ids[i] >= 0 → token, else embedding row i of embd ([n][dim] f32: a host array, or a device tensor
        such as Vision.encode's output)"""
        dim, V = self.model.cfg.dim, self.model.cfg.n_vocab
        ida = None if ids is None else np.ascontiguousarray(ids, dtype=np.int32)
        if embd is None or hasattr(embd, "data_ptr"):
            ea = embd
            n_e = 0 if embd is None else embd.numel() // dim
        else:
            ea = np.ascontiguousarray(embd, dtype=np.float32).reshape(-1, dim)
            n_e = ea.shape[0]
        n = len(ida) if ida is not None else n_e
        out = np.empty(V, np.float32) if logits else None
        _check(lib().ocr_prefill(self.h, slot, _ptr(ida), _ptr(ea), n, _ptr(out)))
        return out

    def step(self, tokens: Sequence[int], logits: bool = True) -> Optional[np.ndarray]:
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        assert t.shape == (self.batch,)
        out = np.empty((self.batch, self.model.cfg.n_vocab), np.float32) if logits else None
        _check(lib().ocr_step(self.h, _ptr(t), _ptr(out)))
        return out

    def decode_gpu(self, slot: int, preset: Preset, history: Sequence[int], max_new: Optional[int] = None,
                   on_token: Optional[Callable[[int], bool]] = None) -> list[int]:
        sc = preset.sampler(max_new)
        h = np.ascontiguousarray(history, dtype=np.int32)
        out = np.empty(sc.max_new, np.int32)
        n = C.c_int(0)
        cb = TOKEN_CB(0) if on_token is None else TOKEN_CB(lambda _u, t: 1 if on_token(int(t)) else 0)
        _check(lib().ocr_decode(self.h, slot, C.byref(sc), _ptr(h) if len(h) else None, len(h), cb, None,
                                _ptr(out), C.byref(n)))
        return out[: n.value].tolist()

    def profile_step(self, tokens: Sequence[int]) -> list[dict]:
        """one eager decode step with an event after every kernel: [{name, layer, us, bytes}] (OCR_WGPU_PROFILE)"""
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        out = (KernelTime * 1024)()
        n = C.c_int(0)
        _check(lib().ocr_profile_step(self.h, _ptr(t), out, 1024, C.byref(n)))
        return [dict(name=out[i].name.decode(), layer=out[i].layer, us=out[i].us, bytes=out[i].bytes)
                for i in range(n.value)]

    def step_embd(self, rows: np.ndarray, active: Optional[Sequence[int]] = None,
                  logits: bool = False) -> Optional[np.ndarray]:
        """one Input::Embeddings row per active slot (rows [batch][dim]), every slot in one step; the logits
        [batch][n_vocab] when asked"""
        r = np.ascontiguousarray(rows, dtype=np.float32).reshape(self.batch, -1)
        act = np.ascontiguousarray(np.ones(self.batch) if active is None else active, dtype=np.int32)
        out = np.empty((self.batch, self.model.cfg.n_vocab), np.float32) if logits else None
        _check(lib().ocr_step_embd(self.h, _ptr(act), _ptr(r), _ptr(out) if logits else None))
        return out

    def timeline_step(self, tokens: Sequence[int], reps: int = 3) -> list[dict]:
        """the in-chain times of one decode step: the step chained as the decode's graph runs it, `reps` times in one
        graph, each launch of the last repetition with the time it adds to the chain ({name, layer, us, bytes})"""
        t = np.ascontiguousarray(tokens, dtype=np.int32)
        out = (KernelTime * 1024)()
        n = C.c_int(0)
        _check(lib().ocr_timeline_step(self.h, _ptr(t), reps, out, 1024, C.byref(n)))
        return [dict(name=out[i].name.decode(), layer=out[i].layer, us=out[i].us, bytes=out[i].bytes)
                for i in range(n.value)]

    def decode_batch(self, preset: Preset, histories: np.ndarray, max_new: Optional[int] = None) -> np.ndarray:
        sc = preset.sampler(max_new)
        h = np.ascontiguousarray(histories, dtype=np.int32).reshape(self.batch, -1)
        out = np.empty((self.batch, sc.max_new), np.int32)
        _check(lib().ocr_decode_batch(self.h, C.byref(sc), _ptr(h) if h.size else None, h.shape[1], _ptr(out)))
        return out


@dataclass
class PageJob:
    """a page for Session.read_pages: prompt rows (token ids and/or embedding rows), the window's start, a budget"""
    id: int
    embd: Optional[np.ndarray]
    max_new: int
    ids: Optional[np.ndarray] = None
    history: Sequence[int] = ()
    out: Optional[np.ndarray] = None  # the chosen ids once read


def read_pages(sess: "Session", preset: Preset, source: Callable[[], Optional[PageJob]],
               on_done: Callable[[PageJob], bool], max_new_cap: int, chunk: int = 16) -> None:
    """ocr_read_pages: pages from `source()` (None = no more) through the session's slots, continuously batched;
    `on_done(page)` gets each read page (page.out = its ids) and returns False to stop"""
    sc = preset.sampler(max_new_cap)
    live: dict[int, tuple] = {}  # page id → (job, the buffers the library reads and writes)

    def _next(_u, pp):
        try:
            job = source()
            if job is None:
                return 0
            dim = sess.model.cfg.dim
            e = None if job.embd is None else np.ascontiguousarray(job.embd, np.float32).reshape(-1, dim)
            ida = None if job.ids is None else np.ascontiguousarray(job.ids, np.int32)
            h = np.ascontiguousarray(job.history, np.int32)
            out = np.zeros(job.max_new, np.int32)
            n = e.shape[0] if e is not None else ida.size
            live[job.id] = (job, e, ida, h, out)
            p = pp.contents
            p.id, p.ids, p.embd, p.n_rows = job.id, _ptr(ida), _ptr(e), n
            p.history, p.n_hist, p.max_new, p.ids_out, p.n_out = _ptr(h) if h.size else None, h.size, job.max_new, \
                _ptr(out), 0
            return 1
        except Exception:  # an exception cannot cross the C ABI: no further page
            import traceback
            traceback.print_exc()
            return 0

    def _done(_u, pp):
        p = pp.contents
        job, _e, _i, _h, out = live.pop(p.id)
        job.out = out[: p.n_out].copy()
        try:
            return 1 if on_done(job) is not False else 0
        except Exception:
            import traceback
            traceback.print_exc()
            return 0

    io = PageIO(None, PAGE_CB(_next), PAGE_CB(_done))
    _check(lib().ocr_read_pages(sess.h, C.byref(sc), chunk, C.byref(io)))


def choose_gpu(ctx: Context, d_logits: int, n_vocab: int, preset: Preset, history: Sequence[int],
               counts: Optional[dict] = None) -> int:
    """ocr_decode::sampling::choose (greedy) on device logits (left unchanged)."""
    sc = preset.sampler(1)
    h = np.ascontiguousarray(history, dtype=np.int32)
    ct = np.ascontiguousarray(list((counts or {}).keys()), dtype=np.int32)
    cn = np.ascontiguousarray(list((counts or {}).values()), dtype=np.uint32)
    tok = np.zeros(1, np.int32)
    _check(lib().ocr_sample_logits(ctx.h, d_logits, n_vocab, C.byref(sc), _ptr(h) if len(h) else None, len(h),
                                   _ptr(ct) if len(ct) else None, _ptr(cn) if len(cn) else None, len(ct), _ptr(tok)))
    return int(tok[0])


# ---------------------------------------------------------------------------------------------------------------------
# low-level ops on device pointers (ints)
# ---------------------------------------------------------------------------------------------------------------------
class Gguf:
    """ocr_gguf::Gguf (host only): header, metadata, tensor infos, small tensors as f32, the text config."""

    def __init__(self, path: Optional[str] = None, data: Optional[bytes] = None):
        h = C.c_void_p()
        if path is not None:
            _check(lib().ocr_gguf_open(str(path).encode(), C.byref(h)))
        else:
            self._buf = C.create_string_buffer(data, len(data)) if data else None
            _check(lib().ocr_gguf_open_memory(self._buf, len(data or b""), C.byref(h)))
        self.h = h

    def close(self) -> None:
        if self.h:
            lib().ocr_gguf_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def header(self) -> dict:
        v, n, a, d = C.c_uint32(), C.c_uint64(), C.c_uint64(), C.c_uint64()
        _check(lib().ocr_gguf_header(self.h, C.byref(v), C.byref(n), C.byref(a), C.byref(d)))
        return dict(version=v.value, n_tensors=n.value, alignment=a.value, data_offset=d.value)

    def u32(self, key: str) -> int:
        v = C.c_uint32()
        _check(lib().ocr_gguf_get_u32(self.h, key.encode(), C.byref(v)))
        return v.value

    def f32(self, key: str) -> float:
        v = C.c_float()
        _check(lib().ocr_gguf_get_f32(self.h, key.encode(), C.byref(v)))
        return v.value

    def str(self, key: str) -> str:
        buf = C.create_string_buffer(4096)
        _check(lib().ocr_gguf_get_str(self.h, key.encode(), buf, 4096))
        return buf.value.decode()

    def f32_array(self, key: str) -> list[float]:
        n = C.c_size_t()
        _check(lib().ocr_gguf_f32_array(self.h, key.encode(), None, 0, C.byref(n)))
        out = np.empty(n.value, np.float32)
        _check(lib().ocr_gguf_f32_array(self.h, key.encode(), _ptr(out), n.value, C.byref(n)))
        return out.tolist()

    def info(self, name: str) -> dict:
        ty, nd, off = C.c_int(), C.c_int(), C.c_uint64()
        shape = (C.c_uint64 * 4)()
        _check(lib().ocr_gguf_tensor(self.h, name.encode(), C.byref(ty), C.byref(shape), C.byref(nd), C.byref(off)))
        return dict(type=ty.value, shape=list(shape)[: nd.value], file_offset=off.value)

    def to_f32(self, name: str) -> np.ndarray:
        n = C.c_size_t()
        _check(lib().ocr_gguf_to_f32(self.h, name.encode(), None, 0, C.byref(n)))
        out = np.empty(n.value, np.float32)
        _check(lib().ocr_gguf_to_f32(self.h, name.encode(), _ptr(out), n.value, C.byref(n)))
        return out

    def text_config(self) -> TextConfig:
        c = TextCfg()
        _check(lib().ocr_gguf_text_config(self.h, C.byref(c)))
        return TextConfig.from_c(c)

    def vision_config(self) -> "VisionConfig":
        """VisionConfig::from_gguf of an mmproj GGUF"""
        c = VisionCfg()
        _check(lib().ocr_gguf_vision_config(self.h, C.byref(c)))
        return VisionConfig(c.n_layer, c.dim, c.n_head, c.n_ff, c.patch, c.merge, c.image_size, c.proj_dim, c.eps,
                            c.rope_theta, tuple(c.mean), tuple(c.std))


def op_penalize(ctx: Context, d_logits: int, n_vocab: int, rp: float, window: int, d_hist: int, n_hist: int) -> None:
    _check(lib().ocr_op_penalize(ctx.h, d_logits, n_vocab, rp, window, d_hist, n_hist))


def q8_row_bytes(cols: int) -> int:
    """the row stride of the device q8_0 layout: int8 quants [cols] | f16 scales [cols/32] | pad to 16 B"""
    return int(lib().ocr_q8_row_bytes(cols))


def q8_rows_from_blocks(blocks: np.ndarray, rows: int, cols: int) -> np.ndarray:
    """GGUF q8_0 blocks → the device row layout, on the host (uint8 [rows][q8_row_bytes(cols)])"""
    stride = (cols + cols // 16 + 15) // 16 * 16
    b = np.asarray(blocks, np.uint8).reshape(rows, cols // 32, 34)
    out = np.zeros((rows, stride), np.uint8)
    out[:, :cols] = b[:, :, 2:].reshape(rows, cols)
    out[:, cols:cols + cols // 16] = b[:, :, :2].reshape(rows, cols // 16)
    return out


def op_repack_q8_0(ctx: Context, d_blocks: int, rows: int, cols: int, d_rows: int) -> None:
    _check(lib().ocr_op_repack_q8_0(ctx.h, d_blocks, rows, cols, d_rows))


def op_matvec_q8_0(ctx: Context, d_w: int, rows: int, cols: int, d_x: int, d_norm_w: Optional[int], eps: float,
                   nb: int, d_y: int, accumulate: bool) -> None:
    _check(lib().ocr_op_matvec_q8_0(ctx.h, d_w, rows, cols, d_x, d_norm_w, eps, nb, d_y, 1 if accumulate else 0))


def op_lm_head_sample(ctx: Context, d_w: int, n_vocab: int, dim: int, d_x: int, d_norm_w: int, eps: float, rp: float,
                      window: int, d_hist: int, d_len: int, d_tok: int, d_logits: Optional[int]) -> None:
    _check(lib().ocr_op_lm_head_sample(ctx.h, d_w, n_vocab, dim, d_x, d_norm_w, eps, rp, window, d_hist, d_len, d_tok,
                                       d_logits))


def op_lm_head_sample_noalloc(ctx: Context, d_w: int, n_vocab: int, dim: int, d_x: int, d_norm_w: int, eps: float,
                              rp: float, window: int, d_hist: int, d_len: int, d_tok: int,
                              d_logits: Optional[int]) -> None:
    """op_lm_head_sample with its scratch in a static device array: the call allocates no device memory"""
    _check(lib().ocr_op_lm_head_sample_noalloc(ctx.h, d_w, n_vocab, dim, d_x, d_norm_w, eps, rp, window, d_hist, d_len,
                                               d_tok, d_logits))


def op_attention_full(ctx: Context, d_q: int, q_stride: int, L: int, n_head: int, d_k_tiled: int, d_vt_tiled: int,
                      n_pad: int, n_keys: int, scale: float, d_out: int, out_stride: int) -> None:
    _check(lib().ocr_op_attention_full(ctx.h, d_q, q_stride, L, n_head, d_k_tiled, d_vt_tiled, n_pad, n_keys, scale,
                                       d_out, out_stride))


def attention_tiles(k: np.ndarray, v: np.ndarray, n_pad: int) -> tuple[np.ndarray, np.ndarray]:
    """K and V [n_head][n][64] (f16) → the vision attention's tiled layouts (ocr_op_attention_full), as uint16"""
    H, n, D = k.shape
    kt = np.zeros((H, n_pad // 64, 64, 64), np.float16)
    vt = np.zeros((H, n_pad // 64, 64, 64), np.float16)
    r = np.arange(64)
    for t0 in range(0, n, 64):
        m = min(64, n - t0)
        kb = np.zeros((H, 64, 64), np.float16)
        vb = np.zeros((H, 64, 64), np.float16)
        kb[:, :m] = k[:, t0:t0 + m]
        vb[:, :m] = v[:, t0:t0 + m]
        for p in range(8):  # key row r, dims 8p … 8p + 7 → piece p ^ (r % 8)
            dst = ((p ^ (r & 7)) * 8)[:, None] + np.arange(8)[None, :]
            kt[:, t0 // 64, r[:, None], dst] = kb[:, :, 8 * p:8 * p + 8]
        vtb = vb.transpose(0, 2, 1)  # [H][dim][key]
        for q in range(8):  # dim row d, keys 8q … 8q + 7 → piece q ^ (d % 8)
            dst = ((q ^ (r & 7)) * 8)[:, None] + np.arange(8)[None, :]
            vt[:, t0 // 64, r[:, None], dst] = vtb[:, :, 8 * q:8 * q + 8]
    return kt.view(np.uint16), vt.view(np.uint16)


# ---------------------------------------------------------------------------------------------------------------------
# a KV cache in fewer bits, attention within a window, trees of drafts (the caller's device memory)
# ---------------------------------------------------------------------------------------------------------------------
KV_TYPES = {"f16": 1, "q4_0": 2, "q8_0": 8}
_KV_ITEM = {1: 2.0, 2: 0.5, 8: 1.0}


def _device_of(t, device: Optional[int] = None) -> int:
    """the GPU that a tensor is on (device: the one it has to be on); the kernels take its address as device memory"""
    try:
        at = t.get_device()
    except AttributeError:
        at = -1
    if at < 0:
        raise OcrError(1, f"the KV operators take device tensors, not {type(t).__name__} in host memory")
    if device is not None and at != device:
        raise OcrError(1, f"a tensor on GPU {at}, its KV cache on GPU {device}")
    return at


class KvCache:
    """A view of one layer's cache (ocr_kv_cache): k, v [n_slot][n_kv][n_rows][row bytes] and, for q8_0 and q4_0, the
    f16 scales [n_slot][n_kv][n_rows][d_head / 32], contiguous device tensors that this view keeps alive. window 0: every
    position is seen; ring: the rows from `sinks` on are used round and round."""

    def __init__(self, type: str, k, v, k_scale=None, v_scale=None, d_head: int = 128, window: int = 0, sinks: int = 0,
                 ring: bool = False):
        if type not in KV_TYPES:
            raise OcrError(1, f"KV cache type {type!r}: one of {', '.join(KV_TYPES)}")
        t = KV_TYPES[type]
        self.device = _device_of(k)
        lead = tuple(k.shape[:3])
        for x, width in ((k, int(d_head * _KV_ITEM[t])), (v, int(d_head * _KV_ITEM[t])), (k_scale, d_head // 16),
                         (v_scale, d_head // 16)):
            if x is None and t == 1:
                continue
            if x is None or tuple(x.shape[:3]) != lead or x.dim() != 4 or not x.is_contiguous() or \
                    x.shape[3] * x.element_size() != width:
                raise OcrError(1, "KV cache tensors must be contiguous [n_slot][n_kv][n_rows][row], rows of d_head")
            _device_of(x, self.device)
        self.c = KvCacheC(t, *lead[:2], d_head, lead[2], window, sinks, int(ring), _ptr(k), _ptr(v),
                          None if t == 1 else _ptr(k_scale), None if t == 1 else _ptr(v_scale))
        self._keep, self._session = (k, v, k_scale, v_scale), None

    @classmethod
    def _of(cls, c: KvCacheC, session: "Session") -> "KvCache":
        v = cls.__new__(cls)
        v.c, v._keep, v._session, v.device = c, (session,), session, session.model.ctx.device
        return v

    def _on(self, ctx: Context) -> KvCacheC:
        """the view for a call on ctx"""
        if self._session is not None and not self._session.h:
            raise OcrError(1, "the session whose rows this KV cache is has been closed")
        if self.device != ctx.device:
            raise OcrError(1, f"the KV cache is on GPU {self.device}, the context on GPU {ctx.device}")
        return self.c

    def nbytes(self) -> tuple[int, int]:
        """the bytes of k (or v) and of k_scale (or v_scale)"""
        return kv_cache_bytes(self.c)


def kv_cache_bytes(c: KvCacheC) -> tuple[int, int]:
    q, s = C.c_size_t(), C.c_size_t()
    _check(lib().ocr_kv_cache_bytes(C.byref(c), C.byref(q), C.byref(s)))
    return q.value, s.value


def rows_of(t, cache: KvCache, heads: Optional[int] = None) -> Rows:
    """a device tensor [n_slot][rows][heads][d_head], f32 or f16, of any strides but the last → ocr_rows"""
    _device_of(t, cache.device)
    shape, stride, item, c = t.shape, t.stride(), t.element_size(), cache.c
    if len(shape) != 4 or shape[0] != c.n_slot or shape[3] != c.d_head or stride[3] != 1 or \
            (heads is not None and shape[2] != heads) or str(t.dtype) not in ("torch.float32", "torch.float16"):
        raise OcrError(1, "rows must be an f32 or f16 tensor [n_slot][rows][heads][d_head], d_head contiguous")
    # (the stride of a dimension of one is anything)
    return Rows(t.data_ptr(), item == 2, stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0,
                stride[2] if shape[2] > 1 else 0)


def _ints(t, cache: KvCache, *shape) -> Optional[int]:
    if t is None:
        return None
    _device_of(t, cache.device)
    if t.shape != shape or str(t.dtype) != "torch.int32" or not t.is_contiguous():
        raise OcrError(1, f"positions, counts, parents and paths are contiguous int32 device tensors, here {list(shape)}")
    return t.data_ptr()


def op_kv_write(ctx: Context, cache: KvCache, k, v, pos, n=None) -> None:
    """rows of keys and values [n_slot][rows][n_kv][d_head] → the cache, from position pos[slot] on (below 0: idle),
    n[slot] of them in use"""
    c = cache._on(ctx)
    if k.shape != v.shape:
        raise OcrError(1, "k and v must be of one shape")
    _check(lib().ocr_op_kv_write(ctx.h, c, rows_of(k, cache, c.n_kv),
                                 rows_of(v, cache, c.n_kv), k.shape[1], _ints(pos, cache, c.n_slot),
                                 _ints(n, cache, c.n_slot)))


def op_kv_read(ctx: Context, cache: KvCache, k, v, pos, n=None) -> None:
    """the cache's rows → values in k and v; rows that are not in use are zeros"""
    c = cache._on(ctx)
    if k.shape != v.shape:
        raise OcrError(1, "k and v must be of one shape")
    _check(lib().ocr_op_kv_read(ctx.h, c, rows_of(k, cache, c.n_kv),
                                rows_of(v, cache, c.n_kv), k.shape[1], _ints(pos, cache, c.n_slot),
                                _ints(n, cache, c.n_slot)))


def op_attention_window(ctx: Context, cache: KvCache, q, out, pos, scale: float, n=None) -> None:
    """rows q [n_slot][rows][n_head][d_head], which the cache already holds from pos[slot] on, attend it: causal, within
    the cache's window and sinks"""
    c = cache._on(ctx)
    if q.shape != out.shape:
        raise OcrError(1, "q and out must be of one shape")
    _check(lib().ocr_op_attention_window(ctx.h, c, rows_of(q, cache), q.shape[2], q.shape[1],
                                         _ints(pos, cache, c.n_slot), _ints(n, cache, c.n_slot), scale, rows_of(out, cache)))


def op_attention_tree(ctx: Context, cache: KvCache, q, out, pos, parent, scale: float, n=None) -> None:
    """the same for a tree of drafts: parent [n_slot][rows], parent[i] < i, -1 for a child of the last committed
    position"""
    c = cache._on(ctx)
    if q.shape != out.shape:
        raise OcrError(1, "q and out must be of one shape")
    _check(lib().ocr_op_attention_tree(ctx.h, c, rows_of(q, cache), q.shape[2], q.shape[1],
                                       _ints(pos, cache, c.n_slot), _ints(n, cache, c.n_slot), _ints(parent, cache, c.n_slot, q.shape[1]),
                                       scale, rows_of(out, cache)))


def op_kv_keep(ctx: Context, caches: Sequence[KvCache], pos, path, n) -> None:
    """the accepted drafts' rows move together in every layer's cache: position pos + path[i] → pos + i, i < n[slot]"""
    cache = caches[0]
    c = cache.c
    rows = path.shape[1]
    arr = (KvCacheC * len(caches))(*[x._on(ctx) for x in caches])
    _check(lib().ocr_op_kv_keep(ctx.h, arr, len(caches), rows, _ints(pos, cache, c.n_slot), _ints(path, cache, c.n_slot, rows),
                                _ints(n, cache, c.n_slot)))


def op_wait_probe(ctx: Context, tries: int) -> bool:
    """runs one device wait that cannot complete, limited to `tries` polls; True when it gave up (the context's error
    flag is then set: the next ctx.sync() raises OcrError with OCR_ERR_DEVICE)"""
    out = C.c_int(0)
    _check(lib().ocr_op_wait_probe(ctx.h, tries, C.byref(out)))
    return bool(out.value)


def op_attention_decode(ctx: Context, d_qkv: int, d_q_norm: int, d_k_norm: int, d_rope: int, d_k: int, d_v: int,
                        n_head: int, n_kv: int, n_ctx: int, pos: int, eps: float, d_out: int) -> None:
    _check(lib().ocr_op_attention_decode(ctx.h, d_qkv, d_q_norm, d_k_norm, d_rope, d_k, d_v, n_head, n_kv, n_ctx,
                                         pos, eps, d_out))


# ---------------------------------------------------------------------------------------------------------------------
# the seeded synthetic data spec (shared with the CPU test generator; numpy, vectorised)
# ---------------------------------------------------------------------------------------------------------------------
_G = np.uint64(0x9E3779B97F4A7C15)
_M1 = np.uint64(0xBF58476D1CE4E5B9)
_M2 = np.uint64(0x94D049BB133111EB)
SEED_BASE = 0x4F43522D42323030  # "OCR-B200"


def splitmix64_at(seed: int, idx: np.ndarray) -> np.ndarray:
    """output idx (0-based) of SplitMix64 seeded with `seed` (ocr-decode sampling.rs:24-35)"""
    with np.errstate(over="ignore"):
        z = np.uint64(seed) + (idx.astype(np.uint64) + np.uint64(1)) * _G
        z = (z ^ (z >> np.uint64(30))) * _M1
        z = (z ^ (z >> np.uint64(27))) * _M2
        return z ^ (z >> np.uint64(31))


def substream(seed: int, k: int) -> int:
    return int(splitmix64_at(seed ^ 0x6F63722D62323030, np.array([k]))[0])


def gauss(seed: int, n: int, sigma: float = 1.0, start: int = 0) -> np.ndarray:
    """sigma * N(0,1) stand-in: Irwin–Hall sum of 12 uniform u16 (3 outputs per value), centred, / 2^16"""
    i = np.arange(start, start + n, dtype=np.uint64)
    s = np.zeros(n, np.int64)
    for k in range(3):
        z = splitmix64_at(seed, np.uint64(3) * i + np.uint64(k))
        for sh in (0, 16, 32, 48):
            s += ((z >> np.uint64(sh)) & np.uint64(0xFFFF)).astype(np.int64)
    g = (s - 6 * 65535).astype(np.float32) * np.float32(1.0 / 65536.0)
    return (np.float32(sigma) * g).astype(np.float32)


def fill_ids(seed: int, n: int, n_vocab: int) -> np.ndarray:
    z = splitmix64_at(seed, np.arange(n, dtype=np.uint64))
    return (((z >> np.uint64(32)) * np.uint64(n_vocab)) >> np.uint64(32)).astype(np.int32)


def version() -> str:
    return lib().ocr_version().decode()
