"""ctypes binding of libdecisioncuda.so (include/decision_cuda.h). Loading fails loudly when the library is
missing: there is no fallback path."""
from __future__ import annotations

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libdecisioncuda.so")

DC_OK, DC_EINVAL, DC_ENOMEM, DC_ECUDA, DC_ETIMEOUT, DC_EFORMAT, DC_EIO = range(7)
ACT_SILU, ACT_GELU_TANH, ACT_GELU_ERF = 0, 1, 2
ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}
K_QGEMM, K_QGEMV, K_ATTN, K_NORM, K_OTHER = range(5)


class DecisionError(RuntimeError):
    """A failed library call: `code` is the DC_E* status, the message starts with "decision.js:" like the
    reference's errors."""

    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


_vp, _i, _f, _d, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_double, ctypes.c_size_t
_SIGS = {
    "dc_last_error": ([], ctypes.c_char_p),
    "dc_init": ([_i, ctypes.POINTER(_vp)], _i),
    "dc_destroy": ([_vp], _i),
    "dc_device_count": ([ctypes.POINTER(_i)], _i),
    "dc_alloc": ([_vp, _sz, ctypes.POINTER(_vp)], _i),
    "dc_free": ([_vp, _vp], _i),
    "dc_upload": ([_vp, _vp, _vp, _sz], _i),
    "dc_download": ([_vp, _vp, _vp, _sz], _i),
    "dc_memset": ([_vp, _vp, _i, _sz], _i),
    "dc_sync": ([_vp, _i], _i),
    "dc_stream": ([_vp], _vp),
    "dc_static_weights": ([_vp, _i], _i),
    "dc_selftest_wait": ([_vp, _i], _i),
    "dc_profile": ([_vp, _i], _i),
    "dc_profile_read": ([_vp, _i, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_longlong),
                         ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)], _i),
    "dc_qmatmul": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i], _i),
    "dc_qmatmul_form": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i], _i),
    "dc_dequant": ([_vp, _vp, _vp, _vp, _i, _i, _i], _i),
    "dc_qmatmul_f16": ([_vp, _vp, _vp, _vp, _i, _i, _i, _i], _i),
    "dc_qmatmul_skinny_noalloc": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i], _i),
    "dc_add_rmsnorm": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _f], _i),
    "dc_sandwich": ([_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _f, _f], _i),
    "dc_qkv_norm_rope": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, _f, _i], _i),
    "dc_attention": ([_vp, _vp, _vp, _vp, _i, _i, _i, _i, _f], _i),
    "dc_attention_form": ([_vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, _i], _i),
    "dc_glu": ([_vp, _vp, _vp, _i, _i, _i], _i),
    "dc_gather": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i], _i),
    "dc_pool": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i], _i),
    "dc_leaf_logits": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _f], _i),
    "dc_short_conv": ([_vp, _vp, _vp, _vp, _vp, _i, _i], _i),
    "dc_ple_mix": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _f], _i),
    "dc_readout": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i], _i),
    "dc_attention_ex": ([_vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, ctypes.c_long, _i, _i], _i),
    "dc_forward_laya": ([_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _i, _vp], _i),
    "dc_forward_omni": ([_vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _i, _vp], _i),
    "dc_forward_d3": ([_vp, _vp, _vp, _vp, _i, _vp, _i, _vp, _i, _vp], _i),
    "dc_gdn": ([_vp, _vp, ctypes.c_long, ctypes.c_long, _i, _vp, _vp, _vp, _vp, _vp, _i, _f, _vp, _i], _i),
    "dc_add_rows": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i], _i),
    "dc_bias_act": ([_vp, _vp, _vp, _i, _i, _i], _i),
    "dc_add_layernorm": ([_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _f], _i),
    "dc_gather_rows": ([_vp, _vp, _vp, _vp, _i, _i, _i], _i),
    "dc_score": ([_vp, _vp, _vp, _vp, _vp, _i, _i], _i),
    "dc_qk_rope": ([_vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, ctypes.c_long, _i, _i, _f, _f], _i),
    "dc_rope_frequencies": ([_i, _d, _i, _d, _d, _d, _d, _vp, _vp], _i),
    "dc_rope_plan_create": ([_vp, _i, _i, _vp, _d, ctypes.POINTER(_vp)], _i),
    "dc_rope_plan_free": ([_vp], _i),
    "dc_rope": ([_vp, _vp, _vp, ctypes.c_long, _vp, _vp, ctypes.c_long, _i, _i, _i], _i),
    "dc_kv_cache_create": ([_vp, _vp, _vp, _i, _i, _i, _i, ctypes.POINTER(_vp)], _i),
    "dc_kv_cache_free": ([_vp], _i),
    "dc_kv_append": ([_vp, _vp, _vp, _vp, ctypes.c_long, _vp, _vp, _f, _i, _vp, _vp, _vp, ctypes.c_long, _i, _i], _i),
    "dc_attention_paged": ([_vp, _vp, _vp, ctypes.c_long, _vp, _i, _vp, _vp, _i, _vp, _i, _vp, _vp, _i, _vp,
                            ctypes.c_long, _i, _i, _f, _vp, _sz], _i),
    "dc_attention_paged_workspace": ([_vp, _vp, _i, _i, _i, _i, ctypes.POINTER(_sz)], _i),
    "dc_load_weights": ([_vp, ctypes.c_char_p, ctypes.POINTER(_vp)], _i),
    "dc_check_weights": ([ctypes.c_char_p], _i),
    "dc_model_free": ([_vp], _i),
    "dc_model_kind": ([_vp, ctypes.c_char_p, _sz], _i),
    "dc_model_config_f": ([_vp, ctypes.c_char_p, ctypes.POINTER(ctypes.c_double)], _i),
    "dc_model_tensor": ([_vp, ctypes.c_char_p, ctypes.POINTER(_vp), ctypes.POINTER(_vp), ctypes.POINTER(_i),
                         ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int64)], _i),
    "dc_forward_encoder": ([_vp, _vp, _vp, _i, _i, _vp], _i),
    "dc_forward_decoder": ([_vp, _vp, _vp, _vp, _i, _vp, _vp, _i, _i, _vp], _i),
    "dc_forward_encoder_device": ([_vp, _vp, _vp, _i, _i, _vp], _i),
    "dc_forward_decoder_device": ([_vp, _vp, _vp, _vp, _i, _vp, _vp, _i, _i, _vp], _i),
    "dc_model_context": ([_vp, ctypes.POINTER(_vp)], _i),
    "dc_eg2_head": ([_vp, _vp, _i, _vp, _i, _vp, _i, _vp, _i, _vp], _i),
}

_lib = None


def lib() -> ctypes.CDLL:
    """The loaded library, with every entry point's signature declared."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise DecisionError(DC_ECUDA, f"decision.js: {LIB_PATH} is not built (run __graft_entry__.build())")
        L = ctypes.CDLL(LIB_PATH)
        for name, (args, res) in _SIGS.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        _lib = L
    return _lib


def symbols() -> list[str]:
    return list(_SIGS)


def check(rc: int) -> None:
    if rc != DC_OK:
        raise DecisionError(rc, lib().dc_last_error().decode() or f"decision.js: error {rc}")


_PLAIN = frozenset((int, float, bool, type(None)))  # arguments that go as they are


def ptr(x) -> int | None:
    """A device or host address from a torch tensor, numpy array, int or None; a handle's from a RopePlan or KvCache."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    address = getattr(x, "data_ptr", None)
    if address is not None:
        return address()
    if hasattr(x, "ctypes"):
        return x.ctypes.data
    raise TypeError(type(x))


def rope_frequencies(rot: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     trained: float = 0.0, a: float | None = None, b: float | None = None):
    """dc_rope_frequencies: (radians per position of each of a head's rot/2 pairs, the factor on cos and sin). `scaling`
    stretches them for a context `factor` times the `trained` one: "none", "linear", "ntk", "yarn" (a, b turns: 32, 1)
    or "bands" (4, 1)."""
    if scaling not in ROPE_SCALINGS:
        raise DecisionError(DC_EINVAL, f"decision.js: rope_frequencies: unknown scaling {scaling!r}")
    a = (32.0 if scaling == "yarn" else 4.0) if a is None else a
    freq = (ctypes.c_double * max(rot // 2, 1))()
    f = ctypes.c_double()
    check(lib().dc_rope_frequencies(rot, theta, ROPE_SCALINGS[scaling], factor, trained, a, 1.0 if b is None else b,
                                    freq, ctypes.byref(f)))
    return list(freq), f.value


def kv_slots(pages, page: int, first: int, count: int) -> list[int]:
    """The cache slots of a sequence's tokens first .. first + count - 1, from its page ids in order."""
    pages = [int(p) for p in pages]
    if first < 0 or count < 0 or first + count > len(pages) * page:
        raise DecisionError(DC_EINVAL, f"decision.js: kv_slots: tokens {first} to {first + count} of {len(pages)} pages "
                                       f"of {page}")
    return [pages[i // page] * page + i % page for i in range(first, first + count)]


class _Handle:
    """A library handle, freed by close() (or with the object)."""

    h = None
    _free = ""

    def data_ptr(self) -> int:
        if not self.h:
            raise DecisionError(DC_EINVAL, f"decision.js: a closed {type(self).__name__}")
        return self.h.value

    def close(self):
        if self.h:
            h, self.h = self.h, None
            check(getattr(lib(), self._free)(h))

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class RopePlan(_Handle):
    """One dc_rope_plan (Context.rope_plan)."""

    _free = "dc_rope_plan_free"

    def __init__(self, h, rot, layout):
        self.h, self.rot, self.layout = h, rot, layout


class KvCache(_Handle):
    """One dc_kv_cache (Context.kv_cache) over k and v, which it keeps alive."""

    _free = "dc_kv_cache_free"

    def __init__(self, h, k, v):
        self.h, self.k, self.v = h, k, v
        self.pages, self.kv, self.page, self.D = k.shape


class Context:
    """One dc_ctx: a CUDA device, its stream and scratch."""

    def __init__(self, device: int = 0):
        h = ctypes.c_void_p()
        check(lib().dc_init(device, ctypes.byref(h)))
        self.h = h
        self.device = device

    def close(self):
        if self.h:
            lib().dc_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def stream(self) -> int:
        return lib().dc_stream(self.h) or 0

    def sync(self, timeout_ms: int = -1):
        check(lib().dc_sync(self.h, timeout_ms))

    def call(self, name: str, *args):
        """Calls dc_<name>(ctx, *args), converting tensors / arrays to addresses, and raises on failure."""
        try:  # (a call's conversions are a good part of its time from the host)
            args = [a if type(a) in _PLAIN else a.data_ptr() for a in args]
        except AttributeError:
            args = [a if isinstance(a, (float, bool, type(None))) else ptr(a) for a in args]
        rc = getattr(lib(), "dc_" + name)(self.h, *args)
        if rc:
            check(rc)

    def rope_plan(self, rot: int, layout: str = "half", frequencies=None, factor: float | None = None, **scaling):
        """A RopePlan for the first `rot` dims of a head, layout "half" or "interleaved": by the given frequencies
        (radians per position, [rot/2]) and factor on cos and sin, or by rope_frequencies(rot, factor=factor, **scaling),
        whose factor is the context's and needs a scaling named."""
        if layout not in ROPE_LAYOUTS:
            raise DecisionError(DC_EINVAL, f"decision.js: rope_plan: unknown layout {layout!r}")
        if frequencies is None:
            if factor is not None:
                if "scaling" not in scaling:
                    raise DecisionError(DC_EINVAL, "decision.js: rope_plan: a factor without frequencies or a scaling")
                scaling["factor"] = factor
            frequencies, factor = rope_frequencies(rot, **scaling)
        elif scaling:
            raise DecisionError(DC_EINVAL, "decision.js: rope_plan: frequencies and a scaling")
        if len(frequencies) != rot // 2:
            raise DecisionError(DC_EINVAL, f"decision.js: rope_plan: {len(frequencies)} frequencies for rot={rot}")
        h = ctypes.c_void_p()
        check(lib().dc_rope_plan_create(self.h, rot, ROPE_LAYOUTS[layout], (ctypes.c_double * max(rot // 2, 1))(*frequencies),
                                        1.0 if factor is None else factor, ctypes.byref(h)))
        return RopePlan(h, rot, layout)

    def kv_cache(self, k, v):
        """A KvCache over two contiguous f16 tensors [pages, kv, page, D] on this context's device."""
        for x in (k, v):
            if x.dim() != 4 or x.shape != k.shape or str(x.dtype) != "torch.float16" or not x.is_contiguous():
                raise DecisionError(DC_EINVAL, "decision.js: kv_cache: k and v are contiguous f16 [pages, kv, page, D]")
        pages, kv, page, D = k.shape
        h = ctypes.c_void_p()
        check(lib().dc_kv_cache_create(self.h, ptr(k), ptr(v), pages, page, kv, D, ctypes.byref(h)))
        return KvCache(h, k, v)

    def attention_paged_workspace(self, cache, T: int, heads: int, S: int, G: int) -> int:
        """The bytes of workspace that dc_attention_paged needs for T rows, S sequences and G groups."""
        n = ctypes.c_size_t()
        check(lib().dc_attention_paged_workspace(self.h, ptr(cache), T, heads, S, G, ctypes.byref(n)))
        return n.value

    def profile(self, enable: bool):
        check(lib().dc_profile(self.h, int(enable)))

    def profile_read(self, kind: int):
        ms, n, fl, by = ctypes.c_double(), ctypes.c_longlong(), ctypes.c_double(), ctypes.c_double()
        check(lib().dc_profile_read(self.h, kind, ctypes.byref(ms), ctypes.byref(n), ctypes.byref(fl),
                                    ctypes.byref(by)))
        return {"ms": ms.value, "launches": n.value, "flops": fl.value, "bytes": by.value}


def device_count() -> int:
    n = ctypes.c_int()
    check(lib().dc_device_count(ctypes.byref(n)))
    return n.value
